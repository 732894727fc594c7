"""How tokens are chosen beside greedily, and where drafted tokens come from.

``Sampling``: one request's temperature, top-k, top-p, min-p and seed (the reference's request parameters, common/data_structures.py:
111-113 there).  Its random number for the token at position p of the sequence is the p-th of its seed's stream, whatever the batch
around it and however many tokens a step makes, and a token follows from its logits and this number alone: the same request gives the same
tokens alone, in a batch, and with drafted tokens, as far as its logits are the same - their sums are rounded in an order that depends on the batch
and on the trees, which in 16 bits moves a token now and then.

``PromptLookup``: drafts from the sequence itself - what followed earlier occurrences of its last tokens, as a tree.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Dict, List, Optional, Sequence, Tuple

import numpy as np


@dataclass(frozen=True)
class Sampling:
    """``temperature`` 0: greedy; ``top_k`` 0, ``top_p`` 1, ``min_p`` 0: no limit; ``seed``: a whole number from 0 on."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if not self.temperature >= 0.0 or self.top_k < 0 or not 0.0 < self.top_p <= 1.0 or not 0.0 <= self.min_p <= 1.0 or self.seed < 0:
            raise ValueError(f"temperature >= 0, top_k >= 0, 0 < top_p <= 1, 0 <= min_p <= 1 and seed >= 0 are wanted: {self}")

    @classmethod
    def of_request(cls, params: Dict[str, Any]) -> "Sampling":
        """From a request's parameters (absent ones and None: their defaults; without a ``seed`` it is 0, the same tokens each time); greedy unless
        it says ``do_sample``.  As other engines write them: ``top_k`` below 0 is no limit, ``seed`` below 0 none, ``top_p`` 0 keeps the likeliest token
        alone."""
        if not params.get("do_sample", False):
            return GREEDY

        def of(name: str, default):
            value = params.get(name)
            return default if value is None else type(default)(value)

        k, p = max(of("top_k", 50), 0), of("top_p", 0.9)
        if p == 0.0:
            k, p = 1, 1.0
        return cls(of("temperature", 0.7), k, p, of("min_p", 0.0), max(of("seed", 0), 0))

    def numbers(self, n: int) -> np.ndarray:
        """The first ``n`` random numbers of the seed's stream, fp32 in [0, 1)."""
        return np.random.Generator(np.random.PCG64(self.seed)).random(n, dtype=np.float32)


GREEDY = Sampling(temperature=0.0)


def settings(rows: Sequence[Sampling]) -> Tuple[np.ndarray, np.ndarray, np.ndarray, np.ndarray]:
    """``(temperature, top_k, top_p, min_p)`` of each row, as ``ops.sample_rows`` takes them."""
    return (np.array([s.temperature for s in rows], np.float32), np.array([min(s.top_k, 2 ** 31 - 1) for s in rows], np.int32),
            np.array([s.top_p for s in rows], np.float32), np.array([s.min_p for s in rows], np.float32))


class PromptLookup:
    """Drafts ``nodes - 1`` tokens at most behind the last one: the continuations of up to ``branches`` earlier occurrences of the sequence's
    last tokens (``longest`` of them if that many occurred before, fewer else), the latest first, joined where they begin alike."""

    def __init__(self, nodes: int = 8, longest: int = 3, branches: int = 2):
        if not 1 <= nodes <= 64 or longest < 1 or branches < 1:
            raise ValueError("1 to 64 nodes, at least one token to look for and one branch")
        self.nodes, self.longest, self.branches = nodes, longest, branches

    def __call__(self, tokens: Sequence[int]) -> Tuple[List[int], List[int]]:
        """``(tokens, parents)`` of the tree's nodes, the root (the last token, parent -1) first."""
        tokens = list(tokens)
        out, parents = [tokens[-1]], [-1]
        ends: List[int] = []
        for n in range(min(self.longest, len(tokens) - 1), 0, -1):
            tail = tokens[-n:]
            for end in range(len(tokens) - 1, n - 1, -1):
                if end not in ends and tokens[end - n:end] == tail:
                    ends.append(end)
                    if len(ends) == self.branches:
                        break
            if len(ends) == self.branches:
                break
        each = -(-(self.nodes - 1) // max(len(ends), 1))
        for end in ends:
            at = 0
            for t in tokens[end:end + each]:
                child = next((i for i in range(at + 1, len(out)) if parents[i] == at and out[i] == t), None)
                if child is None:
                    if len(out) == self.nodes:
                        break
                    child = len(out)
                    out.append(t)
                    parents.append(at)
                at = child
        return out, parents


def pad_trees(trees: Sequence[Optional[Tuple[Sequence[int], Sequence[int]]]], nodes: int):
    """``(tokens int64, parents int32, draft_lens int32)`` of ``[len(trees), nodes]``; None: a sequence without a node."""
    tokens, parents = np.zeros((len(trees), nodes), np.int64), np.full((len(trees), nodes), -1, np.int32)
    lens = np.zeros(len(trees), np.int32)
    for b, tree in enumerate(trees):
        if tree is None:
            continue
        n = len(tree[0])
        if not 1 <= n <= nodes or len(tree[1]) != n or any(not 0 <= p < t for t, p in enumerate(tree[1]) if t > 0):
            raise ValueError(f"a tree of 1 to {nodes} nodes, each behind its parent, is wanted: {tree}")
        tokens[b, :n], parents[b, :n], lens[b] = tree[0], tree[1], n
    return tokens, parents, lens
