"""What the drawing and drafting entry points refuse, without a GPU: Python's checks against a recorder, the C ABI's on null pointers."""
import types

import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import _lib, ops


@pytest.fixture
def recorded(monkeypatch):
    made = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: made.append(name) or 0

    class Guard:
        __enter__ = __exit__ = lambda self, *a: None

    monkeypatch.setattr(ops, "_lib", types.SimpleNamespace(load=Library, check=_lib.check, B200LibraryError=_lib.B200LibraryError))
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_on", lambda device: Guard())
    monkeypatch.setattr(ops, "_tree_workspace", lambda *a: 0)
    return made


def refused(made, call, *changes):
    """`call(**change)` raises ValueError or TypeError and launches nothing; with no change it launches once."""
    call()
    launches = len([n for n in made if not n.endswith("_workspace")])
    assert launches == 1
    for change in changes:
        with pytest.raises((ValueError, TypeError)):
            call(**change)
    assert len([n for n in made if not n.endswith("_workspace")]) == launches


def test_sample_rows(recorded):
    x, u, i = torch.zeros(3, 8), torch.zeros(3), torch.zeros(3, dtype=torch.int32)

    def call(x=x, u=u, **kw):
        return ops.sample_rows(x, u, **kw)

    refused(recorded, call, dict(x=torch.zeros(8)), dict(x=torch.zeros(8, 3).t()), dict(x=x.double()), dict(u=torch.zeros(2)), dict(u=u.double()),
            dict(u=torch.zeros(6)[::2]), dict(temperature=i), dict(temperature=torch.zeros(4)), dict(top_k=u),
            dict(top_k=i.long()), dict(top_p=u.double()), dict(min_p=torch.zeros(3, 1)), dict(out=i), dict(out=torch.zeros(4, dtype=torch.int64)))


def test_draft_tree(recorded):
    par, n = torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def call(par=par, n=n):
        return ops.draft_tree(par, n)

    refused(recorded, call, dict(par=par.long()), dict(par=par[0]), dict(par=torch.zeros(5, 2, dtype=torch.int32).t()), dict(n=n.long()),
            dict(n=torch.zeros(3, dtype=torch.int32)))


def test_paged_tree_attention(recorded):
    i32 = torch.int32
    base = dict(q=torch.zeros(2, 3, 4, 8), k_pool=torch.zeros(5, 2, 16, 8), v_pool=torch.zeros(5, 2, 16, 8), block_tables=torch.zeros(2, 4, dtype=i32),
                context_lens=torch.zeros(2, dtype=i32), visible=torch.zeros(2, 3, dtype=torch.int64))

    def call(**change):
        return ops.paged_tree_attention(**{**base, **change})

    refused(recorded, call, dict(q=torch.zeros(2, 3, 32)), dict(q=torch.zeros(2, 3, 4, 9)), dict(q=base["q"].half()), dict(q=torch.zeros(2, 3, 3, 8)),
            dict(q=torch.zeros(2, 4, 3, 8).transpose(1, 2)), dict(k_pool=base["k_pool"].transpose(1, 2)), dict(v_pool=torch.zeros(5, 2, 16, 16)),
            dict(block_tables=base["block_tables"].long()), dict(block_tables=torch.zeros(3, 4, dtype=i32)), dict(block_tables=torch.zeros(2, 0, dtype=i32)),
            dict(context_lens=torch.zeros(2)), dict(visible=torch.zeros(2, 3, dtype=i32)), dict(visible=torch.zeros(2, 4, dtype=torch.int64)),
            dict(draft_lens=torch.zeros(2)), dict(out=torch.zeros(2, 3, 4, 8).half()), dict(out=torch.zeros(2, 3, 4, 16)[..., ::2]))


def test_accept_drafts(recorded):
    i32, i64 = torch.int32, torch.int64
    base = dict(tokens=torch.zeros(2, 3, dtype=i64), chosen=torch.zeros(2, 3, dtype=i64), parents=torch.zeros(2, 3, dtype=i32),
                visible=torch.zeros(2, 3, dtype=i64), k_ptrs=torch.zeros(4, dtype=i64), v_ptrs=torch.zeros(4, dtype=i64), pool_shape=(5, 2, 16, 8),
                dtype=torch.float32, block_tables=torch.zeros(2, 4, dtype=i32), context_lens=torch.zeros(2, dtype=i32))

    def call(**change):
        return ops.accept_drafts(**{**base, **change})

    refused(recorded, call, dict(tokens=base["tokens"].int()), dict(tokens=base["tokens"][0]), dict(chosen=torch.zeros(2, 4, dtype=i64)),
            dict(parents=base["parents"].long()), dict(visible=base["visible"].int()), dict(k_ptrs=None), dict(v_ptrs=torch.zeros(3, dtype=i64)),
            dict(k_ptrs=torch.zeros(4, dtype=i32)), dict(block_tables=torch.zeros(2, 4)), dict(context_lens=torch.zeros(3, dtype=i32)),
            dict(draft_lens=torch.zeros(2, dtype=i64)))


def test_the_library_refuses():
    lib = _lib.load()

    def says(rc, code, text):
        assert rc == code and text in lib.b200_last_error()

    says(lib.b200_sample_rows(None, None, 2, 8, 8, None, None, 1.0, None, 0, None, 1.0, None, 0.0, 7, None), -1, b"unsupported dtype")
    says(lib.b200_sample_rows(None, None, 2, 8, -1, None, None, 1.0, None, 0, None, 1.0, None, 0.0, 2, None), -1, b"bad sizes")
    says(lib.b200_sample_rows(None, None, 2, 8, 8, None, None, 1.0, None, 0, None, 1.0, None, 0.0, 2, None), -1, b"null pointer")
    says(lib.b200_sample_rows(None, None, 2, (1 << 20) + 1, 1 << 21, None, None, 1.0, None, 0, None, 1.0, None, 0.0, 2, None), -2, b"rows of")
    assert lib.b200_sample_rows(None, None, 0, 8, 8, None, None, 1.0, None, 0, None, 1.0, None, 0.0, 2, None) == 0
    says(lib.b200_draft_tree(None, None, None, 3, None, 2, 65, None), -2, b"at most 64")
    says(lib.b200_draft_tree(None, None, None, 3, None, 2, 3, None), -1, b"null pointer")
    attn = lambda nodes=3, hq=4, hkv=2, dtype=2, cols=4: lib.b200_paged_tree_attn(  # noqa: E731
        None, None, 0, 0, None, None, None, 4, cols, None, None, None, 3, 2, nodes, hq, hkv, 64, 16, 10, 1.0, None, 0, dtype, 0, None)
    says(attn(nodes=65), -2, b"at most 64")
    says(attn(hq=5), -2, b"multiple")
    says(attn(dtype=9), -1, b"unsupported dtype")
    says(attn(cols=0), -1, b"bad sizes")
    says(attn(), -1, b"null pointer")
    accept = lambda nodes=3, layers=2, dtype=2: lib.b200_accept_drafts(  # noqa: E731
        None, None, None, None, None, 3, None, 3, None, 3, None, 3, None, None, layers, None, 4, 4, None, None, 2, nodes, 2, 64, 16, 10, dtype, None)
    says(accept(nodes=65), -2, b"at most 64")
    says(accept(dtype=5), -1, b"unsupported dtype")
    says(accept(layers=40000), -2, b"layers")
    says(accept(), -1, b"null pointer")


def test_tensors_of_several_devices(recorded, monkeypatch):
    """Devices by their numbers, as a GPU box has them."""
    other = torch.zeros(3)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1 if t.data_ptr() == other.data_ptr() else 0)
    x, u = torch.zeros(3, 8), torch.zeros(3)
    ops.sample_rows(x, u, u)
    for kw in (dict(u=other), dict(u=u, temperature=other), dict(u=u, top_p=other), dict(u=u, min_p=other)):
        with pytest.raises(ValueError):
            ops.sample_rows(x, **kw)
    assert recorded == ["b200_sample_rows"]


def test_no_cpu_form():
    with pytest.raises(_lib.B200LibraryError):
        ops.sample_rows(torch.zeros(1, 4), torch.zeros(1))
    with pytest.raises(_lib.B200LibraryError):
        ops.draft_tree(torch.zeros(1, 4, dtype=torch.int32))


def test_sampling_settings():
    from dgi_b200.drafting import GREEDY, Sampling, settings

    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2.0), dict(seed=-1)):
        with pytest.raises(ValueError):
            Sampling(**bad)
    assert Sampling.of_request({"temperature": 0.3}) == GREEDY
    assert Sampling.of_request({"do_sample": True}) == Sampling(0.7, 50, 0.9, 0.0, 0)
    assert Sampling.of_request({"do_sample": True, "temperature": 1, "top_k": 0, "top_p": 1, "min_p": 0.1, "seed": 4}) == Sampling(1.0, 0, 1.0, 0.1, 4)
    assert Sampling.of_request({"do_sample": True, "temperature": None, "top_k": None, "top_p": None, "min_p": None, "seed": None}) == Sampling(0.7, 50, 0.9)
    t, k, p, m = settings([GREEDY, Sampling(0.5, 7, 0.9, 0.1)])
    assert t.tolist() == [0.0, 0.5] and k.tolist() == [0, 7] and abs(p[1] - 0.9) < 1e-6 and abs(m[1] - 0.1) < 1e-6
    a = Sampling(seed=3).numbers(100)
    assert (a[:40] == Sampling(seed=3).numbers(40)).all() and (a >= 0).all() and (a < 1).all() and (a != Sampling(seed=4).numbers(100)).any()


def test_prompt_lookup_and_padding():
    from dgi_b200.drafting import PromptLookup, pad_trees

    look = PromptLookup(nodes=6, longest=2, branches=2)
    assert look([5]) == ([5], [-1]) and look([1, 2, 3]) == ([3], [-1])
    # "1 2" was followed by 3 4 and, before, by 3 9: one branch to 3, then two of two tokens
    assert look([1, 2, 3, 9, 1, 2, 3, 4, 1, 2]) == ([2, 3, 4, 1, 9, 1], [-1, 0, 1, 2, 1, 4])
    tokens, parents = look(list(range(20)) * 3)
    assert len(tokens) <= 6 and tokens[0] == 19 and all(0 <= p < t for t, p in enumerate(parents) if t)
    for bad in (dict(nodes=0), dict(nodes=65), dict(longest=0), dict(branches=0)):
        with pytest.raises(ValueError):
            PromptLookup(**bad)
    t, p, n = pad_trees([([4, 5], [-1, 0]), None], 3)
    assert t.tolist() == [[4, 5, 0], [0, 0, 0]] and p.tolist() == [[-1, 0, -1], [-1, -1, -1]] and n.tolist() == [2, 0]
    for bad in (([1, 2], [-1, 1]), ([1, 2], [-1]), ([], []), ([1] * 4, [-1, 0, 0, 0])):
        with pytest.raises(ValueError):
            pad_trees([bad], 3)
