"""Decoding over a cache in 8 bits: the engine with the kernels against the engine with their definitions in elementary torch, and against itself."""
import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import ops
from dgi_b200.engine import PagedDecodeEngine
from dgi_b200.testing import build_product_shards
from dgi_b200.worker.engines.paged_engine import PagedLLMEngine
from oracle import llama_ref as L
from test_q8_cache_gpu import attention_reference, write_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = ("int8", "e4m3")


def model(golden, dtype=torch.float32, ranges=((0, 2), (2, 4))):
    g = golden("tiny_decode.json")
    cfg = L.RefConfig(**g["config"])
    return g, cfg, build_product_shards(cfg, L.make_weights(cfg, seed=0), list(ranges), device=DEV, dtype=dtype)


class Definitions:
    """The four entry points by their definitions; what each call was given goes to `calls`."""

    def __init__(self):
        self.calls = []

    def rope_kv_append_q8(self, q, k, v, cos, sin, k_pool, v_pool, k_scale, v_scale, tables, lens, row_starts=None, max_new=None, q_out=None):
        self.calls.append("write")
        starts = list(range(len(lens) + 1)) if row_starts is None else row_starts.tolist()
        for to, new in zip((k_pool, v_pool, k_scale, v_scale),
                           write_reference(k, v, cos, sin, k_pool, v_pool, k_scale, v_scale, tables, lens.tolist(), starts)):
            (to if to.dtype == torch.float32 else to.view(torch.uint8)).copy_(new if to.dtype == torch.float32 else new.view(torch.uint8))
        D = q.shape[2]
        x, c, s = q.float(), cos.float()[:, None], sin.float()[:, None]
        return (x * c + torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1) * s).to(q.dtype)

    def _attention(self, q, k_pool, v_pool, k_scale, v_scale, tables, lens, starts):
        return attention_reference(q, k_pool, v_pool, k_scale, v_scale, tables, lens.tolist(), starts, q.shape[2] ** -0.5, False)[0].to(q.dtype)

    def paged_decode_attention_q8(self, q, k_pool, v_pool, k_scale, v_scale, tables, lens, longest, flags=0):
        self.calls.append("decode")
        return self._attention(q, k_pool, v_pool, k_scale, v_scale, tables, lens, list(range(len(lens) + 1)))

    def paged_prompt_attention_q8(self, q, k_pool, v_pool, k_scale, v_scale, tables, lens, starts, most, longest, flags=0):
        self.calls.append("prompt")
        return self._attention(q, k_pool, v_pool, k_scale, v_scale, tables, lens, starts.tolist())

    def kv_gather_dense_q8(self, k_pool, v_pool, k_scale, v_scale, tables, n, dtype):
        self.calls.append("read")
        bs = k_pool.shape[2]
        at, t = tables.long()[:, torch.arange(n, device=DEV) // bs], torch.arange(n, device=DEV) % bs
        return tuple((p.view(torch.uint8)[at, :, t].view(p.dtype).float() * s[at][..., None]).transpose(1, 2).to(dtype) for p, s in ((k_pool, k_scale), (v_pool, v_scale)))


def logits_of(eng, prompts, tokens):
    """Logits of the prompts' last tokens and of given tokens behind them, one step after the other."""
    eng.allocate(prompts.shape[0], prompts.shape[1] + tokens.shape[1] + 1)
    eng.logits_log = []
    eng.prefill(prompts)
    for t in range(tokens.shape[1]):
        eng.decode_step(tokens[:, t])
    rows = [None] * prompts.shape[0]
    steps = []
    for lo, hi, x in eng.logits_log:
        for b in range(lo, hi):
            rows[b] = x[b - lo]
        if hi == prompts.shape[0]:
            steps.append(torch.stack(rows))
    return torch.stack(steps)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mode", ["sdpa", "eager"])
@pytest.mark.parametrize("fused", [False, True])
def test_the_engine_calls_the_operators(golden, monkeypatch, kind, mode, fused):
    """fp32: logits as with the definitions in the kernels' places.  A number that falls next to the border of two codes may take the other (a 2^-24 off of 127
    steps: one in 10^5), which moves an output by a step of one key's channel at most, 1 / 127 of the page's largest times that key's weight: 1e-3 of the logits' size
    is above all that."""
    g, cfg, shards = model(golden)
    prompts, tokens = torch.tensor(g["prompt_ids"]), torch.tensor(g["tokens"])[:, :20]
    eng = PagedDecodeEngine(shards, 4, 192, prefill_mode=mode, use_cuda_graph=False, kv_cache_dtype=kind, fuse_projections=fused)
    got = logits_of(eng, prompts, tokens)
    plain = Definitions()
    for name in ("rope_kv_append_q8", "paged_decode_attention_q8", "paged_prompt_attention_q8", "kv_gather_dense_q8"):
        monkeypatch.setattr(ops, name, getattr(plain, name))
    want = logits_of(eng, prompts, tokens)
    assert {"write", "decode", "read" if mode == "eager" else "prompt"} == set(plain.calls)
    assert ((got - want).norm() / want.norm()).item() < 1e-3


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graphs_replay_what_launches_do(golden, kind, dtype):
    g, cfg, shards = model(golden, dtype)
    prompts = torch.tensor(g["prompt_ids"])
    a = PagedDecodeEngine(shards, 4, 192, kv_cache_dtype=kind)
    b = PagedDecodeEngine(shards, 4, 192, use_cuda_graph=False, kv_cache_dtype=kind)
    first = a.generate(prompts, 40)
    assert torch.equal(first, b.generate(prompts, 40))
    assert torch.equal(first[:2], a.generate(prompts[:2], 40)) or dtype != torch.float32     # (16 bits: other batches have other products)
    assert torch.equal(first, a.generate(prompts, 40)), "blocks that other sequences had before"
    # steps that stay on the device
    a.allocate(4, prompts.shape[1] + 40)
    told = [a.prefill(prompts)]
    a.ids_buf[:4, 0].copy_(told[0])
    for _ in range(39):
        a.decode_step_device()
        told.append(a.next_tokens[:4].clone())
    assert torch.equal(torch.stack(told, 1).cpu(), first)


def test_pools_take_a_byte_a_number_and_blocks_are_shared(golden):
    g, cfg, shards = model(golden, torch.bfloat16)
    prompts = torch.tensor(g["prompt_ids"])
    prompts = torch.cat((prompts[:1, :48].expand(4, -1), prompts), 1)      # a system prompt of three blocks
    eng = PagedDecodeEngine(shards, 4, 256, kv_cache_dtype="int8", prefix_cache=True, spare_blocks=16)
    full = PagedDecodeEngine(shards, 4, 256)
    assert all(p.backing.element_size() == 1 and 2 * p.backing.numel() * p.backing.element_size() == q.backing.numel() * q.backing.element_size() * p.max_blocks_per_layer
               // q.max_blocks_per_layer for p, q in zip(eng.pools, full.pools))
    alone = eng.generate(prompts, 8)
    shared = eng.generate(prompts, 8, shared_prefix_len=48)
    assert eng.cached_blocks == 0 and len({tuple(eng.block_tables[b, :3].tolist()) for b in range(4)}) == 1
    again = eng.generate(prompts, 8, shared_prefix_len=48)
    assert eng.cached_blocks == 3
    assert alone.shape == shared.shape and torch.equal(shared[1:], again[1:])       # (the first sequence's own tokens now come as a portion of their own)


def test_ragged_prompts_and_requests(golden):
    g, cfg, shards = model(golden)
    prompts = [p[:n] for p, n in zip(g["prompt_ids"], (5, 17, 33, 40))]
    eng = PagedDecodeEngine(shards, 4, 192, kv_cache_dtype="int8")
    got = eng.generate_ragged(prompts, 12)
    for p, t in zip(prompts, got):
        assert eng.generate(torch.tensor([p]), 12).tolist() == [t]
    answers = eng.batch_inference([dict(input_ids=p, max_new_tokens=12) for p in prompts])
    assert [a["output_ids"] for a in answers] == got


def test_the_engine_surface_takes_it(golden):
    g, cfg, shards = model(golden)
    e = PagedLLMEngine(dict(shards=shards, max_batch_size=4, max_model_len=192, kv_cache_dtype="e4m3", prefix_cache_blocks=8))
    e.load_model()
    assert e.engine.kv_cache_dtype == "e4m3" and e.engine.pools[0].backing.element_size() == 1
    out = e.inference(dict(input_ids=g["prompt_ids"][0], max_tokens=6))
    assert out["usage"]["completion_tokens"] == 6


def test_refusals(golden):
    g, cfg, shards = model(golden)
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        PagedDecodeEngine(shards, 2, 64, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="kv_pools"):
        PagedDecodeEngine(shards, 2, 64, kv_cache_dtype="int8", kv_pools=PagedDecodeEngine(shards, 2, 64).pools)
    eng = PagedDecodeEngine(shards, 2, 64, kv_cache_dtype="int8")
    prompts = torch.tensor(g["prompt_ids"])[:2, :20]
    with pytest.raises(RuntimeError, match="8 bits"):
        eng.generate_drafted(prompts, 4)
    eng.allocate(2, 40)
    eng.prefill(prompts)
    with pytest.raises(RuntimeError, match="8 bits"):
        eng.verify_trees(torch.zeros(2, 1, dtype=torch.int64), torch.full((2, 1), -1, dtype=torch.int32))
