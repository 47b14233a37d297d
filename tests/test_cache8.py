"""The paged 8-bit cache's and the log probabilities' entries without a GPU: what they refuse before any launch (no
call here reaches one), and the attention's scratch sizes."""
import ctypes

import pytest

from b200fwd import abi
from conftest import ROOT

P = 1 << 20  # a pointer that no refused call follows, on every alignment


@pytest.fixture(scope="module")
def lib():
    import sys

    sys.path.insert(0, str(ROOT / "pyodide-llm_b200"))
    import build

    build.build()
    return abi.load()


TABLES = dict(tables=P, ring=P, state_out=P, lengths_out=P, starts=P, slots=P, seq=P, pos=P, state=P, lengths=P, news=P,
              n_seqs=4, table_width=8, blocks=32, block=16, n=8, stream=None)
STORE = dict(kc=P, ks=P, vc=P, vs=P, k=P, v=P, slots=P, n=4, k_stride=128, v_stride=128, blocks=8, block=16, nkv=2, hs=64,
             half=0, stream=None)
ATTENTION = dict(out=P, q=P, kc=P, ks=P, vc=P, vs=P, tables=P, starts=P, lengths=P, n=4, n_seqs=2, table_width=4, blocks=8,
                 block=16, nh=4, nkv=2, hs=64, q_stride=256, out_stride=256, half=0, scratch=P, stream=None)
LOGPROBS = dict(logprob=P, entropy=P, top_logprob=P, top_id=P, logits=P, targets=P, count=2, n=100, stride=100, k=5, half=0,
                stream=None)


def refused(fn, base, change, words):
    rc = fn(*{**base, **change}.values())
    assert rc == abi.EINVAL
    assert words in abi.last_error(), abi.last_error()


@pytest.mark.parametrize("change,words", [
    ({"tables": None}, "null"), ({"ring": None}, "null"), ({"slots": None}, "null"), ({"news": None}, "null"),
    ({"n_seqs": 0}, "requests"), ({"n_seqs": 1 << 21}, "requests"), ({"n": -1}, "tokens"), ({"block": 8}, "16 positions"),
    ({"block": 24}, "16 positions"), ({"block": 512}, "16 positions"), ({"blocks": 0}, "1 block"),
    ({"blocks": 1 << 28}, "int32"), ({"table_width": 0}, "1 block"), ({"table_width": 1 << 28}, "int32"),
])
def test_block_tables_refusals(lib, change, words):
    refused(lib.b200k_block_tables, TABLES, change, words)


@pytest.mark.parametrize("entry", ["store", "load"])
@pytest.mark.parametrize("change,words", [
    ({"kc": None}, "null"), ({"vs": None}, "null"), ({"k": None}, "null"), ({"slots": None}, "null"), ({"n": -1}, "tokens"),
    ({"n": (1 << 30) + 1}, "tokens"), ({"k_stride": 127}, "stride"), ({"v_stride": 130}, "16 bytes"),
    ({"half": 1, "k_stride": 132}, "16 bytes"), ({"k": P + 4}, "16 bytes"), ({"kc": P + 8}, "aligned"),
    ({"block": 40}, "16 positions"), ({"hs": 24}, "head size"), ({"hs": 272}, "head size"), ({"nkv": 0}, "kv heads"),
    ({"nkv": 1025}, "kv heads"), ({"blocks": 0}, "1 block"), ({"blocks": 1 << 28}, "int32"),
])
def test_cache8_rows_refusals(lib, entry, change, words):
    if entry == "store":
        refused(lib.b200k_cache8_store, STORE, change, words)
    else:
        order = ("k", "v", "kc", "ks", "vc", "vs")
        refused(lib.b200k_cache8_load, {**{x: STORE[x] for x in order}, **STORE}, change, words)


@pytest.mark.parametrize("change,words", [
    ({"out": None}, "null"), ({"scratch": None}, "null"), ({"kc": None}, "null"), ({"starts": None}, "null"),
    ({"n": -1}, "tokens"), ({"n_seqs": 0}, "requests"), ({"n_seqs": 65537}, "requests"), ({"nh": 5}, "multiple"),
    ({"nh": 1}, "multiple"), ({"nkv": 0}, "multiple"), ({"hs": 72}, "head size"), ({"hs": 512}, "head size"),
    ({"block": 0}, "16 positions"), ({"q_stride": 255}, "rows"), ({"out_stride": 258}, "rows"), ({"q": P + 8}, "rows"),
    ({"half": 1, "q_stride": 260}, "rows"), ({"scratch": P + 16}, "256-byte"), ({"table_width": 0}, "table row"),
    ({"table_width": 1 << 27}, "table row"), ({"n": 1 << 29}, "2^30"),
])
def test_cache8_attention_refusals(lib, change, words):
    refused(lib.b200k_cache8_attention, ATTENTION, change, words)


def test_cache8_attention_scratch(lib):
    size = ctypes.c_uint64()
    assert lib.b200k_cache8_attention_scratch(64, 64, 32, 8, 128, 0, ctypes.byref(size)) == 0
    one = size.value
    assert 0 < one < 64 << 20  # partial sums of a step of 64 requests
    assert lib.b200k_cache8_attention_scratch(4096, 64, 32, 8, 128, 0, ctypes.byref(size)) == 0
    assert size.value > one
    assert lib.b200k_cache8_attention_scratch(4, 4, 5, 2, 64, 0, ctypes.byref(size)) == abi.EINVAL
    assert lib.b200k_cache8_attention_scratch(4, 4, 4, 2, 64, 0, None) == abi.EINVAL


def test_calls_of_no_tokens_do_nothing(lib):
    """n = 0 returns before any launch (there may be no GPU)."""
    assert lib.b200k_cache8_store(*{**STORE, "n": 0}.values()) == 0
    assert lib.b200k_cache8_attention(*{**ATTENTION, "n": 0}.values()) == 0
    assert lib.b200k_logprobs(*{**LOGPROBS, "count": 0}.values()) == 0


@pytest.mark.parametrize("change,words", [
    ({"logits": None}, "null"), ({"targets": None}, "null"), ({"top_id": None}, "null"), ({"top_logprob": None}, "null"),
    ({"count": -1}, "rows"), ({"n": 0}, "logits"), ({"stride": 99}, "stride"), ({"k": 33}, "alternatives"),
    ({"k": -1}, "alternatives"), ({"n": 4, "k": 5}, "alternatives"), ({"logits": P + 2}, "misaligned"),
    ({"half": 1, "logits": P + 1}, "misaligned"),
])
def test_logprobs_refusals(lib, change, words):
    refused(lib.b200k_logprobs, LOGPROBS, change, words)
