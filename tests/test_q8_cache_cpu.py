"""CPU: what the entry points of the cache in 8 bits refuse before anything is launched."""
import os
import re
import subprocess
import sysconfig

import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import _lib, ops


def test_host_tensors_are_refused():
    pool, scale = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2)
    tables, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.paged_decode_attention_q8(q, pool, pool, scale, scale, tables, lens, 16),
                 lambda: ops.paged_prompt_attention_q8(q, pool, pool, scale, scale, tables, lens, torch.zeros(2, dtype=torch.int32), 1, 16),
                 lambda: ops.kv_gather_dense_q8(pool, pool, scale, scale, tables, 4),
                 lambda: ops.kv_append_q8(q[:, :2], q[:, :2], pool, pool, scale, scale, tables, lens)):
        with pytest.raises(_lib.B200LibraryError):
            call()


def test_argument_errors_have_codes_and_words():
    lib = _lib.load()
    p = 4096      # never read: every call below is refused

    def append(**over):
        a = dict(out=p, os=512, q=p, qs=512, k=p, ks=256, v=p, vs=256, cos=p, sin=p, kp=p, vp=p + 16, s=p, t=p + 16, table=p, stride=4, cols=4, lens=p, starts=p, B=2, rows=5,
                 most=5, Hq=4, Hkv=2, D=128, bs=16, blocks=8, codes=3, dtype=2, stream=None)
        a.update(over)
        return lib.b200_rope_kv_append_q8(*a.values()), lib.b200_last_error().decode()

    def prompt(**over):
        a = dict(out=p, q=p, qs=512, kp=p, vp=p, s=p, t=p, table=p, stride=4, cols=4, lens=p, starts=p, B=2, rows=5, most=5, Hq=4, Hkv=2, D=128, bs=16, blocks=8,
                 scale=1.0, longest=64, ws=None, bytes=0, codes=3, dtype=2, flags=0, stream=None)
        a.update(over)
        return lib.b200_paged_prompt_attn_q8(*a.values()), lib.b200_last_error().decode()

    def decode(**over):
        a = dict(out=p, q=p, qs=512, kp=p, vp=p, s=p, t=p, table=p, stride=4, cols=4, lens=p, B=2, Hq=4, Hkv=2, D=128, bs=16, blocks=8, scale=1.0, longest=64, ws=None,
                 bytes=0, codes=3, dtype=2, flags=0, stream=None)
        a.update(over)
        return lib.b200_paged_decode_attn_q8(*a.values()), lib.b200_last_error().decode()

    def gather(**over):
        a = dict(k=p, v=p, kp=p, vp=p, s=p, t=p, table=p, stride=4, cols=4, B=2, n=40, Hkv=2, D=128, bs=16, blocks=8, codes=3, dtype=2, stream=None)
        a.update(over)
        return lib.b200_kv_gather_dense_q8(*a.values()), lib.b200_last_error().decode()

    for call in (append, prompt, decode, gather):
        for over, words in ((dict(dtype=7), "dtype"), (dict(codes=5), "codes"), (dict(D=0), "sizes"), (dict(bs=0), "sizes"), (dict(blocks=0), "sizes"),
                            (dict(blocks=2 ** 31), "sizes"), (dict(cols=0), "sizes"), (dict(B=-1), "sizes"), (dict(kp=None), "null"), (dict(t=None), "null")):
            rc, said = call(**over)
            assert rc == -1 and words in said, (call.__name__, over, rc, said)
        assert call(B=0)[0] == 0
    for call in (prompt, decode):
        assert call(Hq=5)[0] == -2 and call(longest=-1)[0] == -1 and call(D=512)[0] == -2 and call(out=None)[0] == -1
    assert prompt(rows=0)[0] == 0 and prompt(starts=None)[0] == -1 and prompt(most=-1)[0] == -1
    assert decode(longest=4096, dtype=0)[0] == -3
    assert append(rows=0)[0] == 0 and append(starts=None)[0] == -1 and append(sin=None)[0] == -1 and append(cos=None, sin=None)[0] == -1
    assert append(D=33)[0] == -2 and append(q=None)[0] == -1 and append(B=2 ** 30, most=2 ** 30, rows=2 ** 30)[0] == -2
    assert append(vp=p)[0] == -1 and append(t=p)[0] == -1
    assert gather(n=65)[0] == -1 and gather(n=0)[0] == 0


def test_the_fast_module_leaves_what_is_not_plain_to_the_checks():
    fast = _lib.fast_calls()
    assert fast is not None, "the module of fast calls is not built: run __graft_entry__.build()"
    pool, scale = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2)
    tables, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    cache = (pool, pool, scale, scale, tables)
    for got in (fast.decode(q, *cache, lens, 16, None), fast.decode(q, *cache, lens), fast.decode(), fast.decode(None, *cache, lens, 16, 0.5),
                fast.prompt(q, *cache, lens, lens, 1, 16, None), fast.prompt(1, 2, 3), fast.gather(*cache, 4, 2), fast.gather(*cache, "4", None),
                fast.append(q, q, q, q[0], q[0], *cache, lens, None, None), fast.append(None)):
        assert got is None
    with pytest.raises(TypeError):
        fast.entry_points(1, 2)
    with pytest.raises(ValueError):
        fast.entry_points(1, 2, 3, 4, 5, 0)


ODD_PARTS = [(1, 1301, 9, 3, 64, 1301), (3, 101, 5, 1, 128, 1301), (1, 207, 5, 1, 128, 2255), (9, 127, 1, 1, 128, 1400), (1, 205, 5, 1, 128, 1434), (1, 801, 5, 1, 128, 4801),
             (5, 193, 1, 1, 64, 1410), (23, 33, 1, 1, 64, 2300), (5, 33, 3, 1, 128, 20033)]


@pytest.mark.parametrize("B,new,Hq,Hkv,D,longest", ODD_PARTS + [(1, 206, 5, 1, 128, 2255), (2, 105, 5, 1, 64, 1301), (3, 101, 4, 2, 128, 1301)])
def test_outputs_of_parts_begin_at_a_multiple_of_16_bytes(B, new, Hq, Hkv, D, longest):
    """The workspace of several tokens in parts: statistics of 8 bytes for each row and part, brought to whole 16 bytes, then the parts' outputs, stored 16 bytes at once."""
    lib = _lib.load()
    for block_size in (16, 48):
        need = lib.b200_paged_prompt_attn_q8_workspace(B, new, Hq, Hkv, D, block_size, longest, 2)
        rows = B * new * Hq
        parts = need // (rows * (8 + 4 * D))
        n = rows * parts
        assert parts > 1 and (n % 2 == 1) == ((B, new, Hq, Hkv, D, longest) in ODD_PARTS), parts
        assert need == (n + 1) // 2 * 16 + n * D * 4


@pytest.mark.parametrize("name,kernels", [("b200_kv_q8.cu", ("append_kernel", "gather_kernel")), ("b200_attn_q8.cu", ("decode_merge_kernel",)), ("b200_prompt_q8.cu", ("prompt_merge_kernel",))])
def test_kernels_that_begin_beside_the_one_ahead_read_coherently(name, kernels):
    """They are there while the kernel ahead writes what they read: none of their loads may be of the kind for memory that nobody writes meanwhile (ld.global.nc)."""
    with open(os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc", name)) as f:
        source = f.read()
    for kernel in kernels:
        body = re.search(r"__global__[^;{]*\b" + kernel + r"\(.*?\n}\n", source, re.S).group(0)
        assert "griddepcontrol.wait" in body or "wait_for_ahead()" in body
        assert not re.search(r"\.nc\b|\bld_stream\w*\(|__ldg\(|__ldcs\(", body), kernel


def test_the_libraries_build_without_a_python_that_has_torch():
    csrc = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    done = subprocess.run(["make", "-C", csrc, "all", "PYTHON=false", "-o", "../libb200_kv.so", "-o", "../libb200_mixers.so", "-W", "b200_fast_calls.cpp"],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, stdin=subprocess.DEVNULL, timeout=120)
    assert done.returncode == 0, done.stdout.decode()


def test_the_fast_module_is_of_this_interpreter_and_this_torch(monkeypatch):
    name = os.path.basename(_lib.fast_calls().__file__)
    assert torch.__version__ in name and sysconfig.get_config_var("SOABI") in name
    monkeypatch.setattr(_lib, "_fast", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert _lib.fast_calls() is None
