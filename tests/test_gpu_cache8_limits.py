"""Where the paged 8-bit cache and its attention can go wrong: queries and keys of zeros, queries of any size, scales at
float32's lower end, starts that do not ascend, outliers among a query's values, weights far below the largest one, and
requests of more steps than the prompt kernel's rings hold. GPU only."""
import ctypes

import numpy as np
import pytest
import torch

from b200fwd import abi
from gpu_util import full, host, ptr
from test_gpu_cache8 import Case, store_case

pytestmark = pytest.mark.gpu

# more than 64 rows a kv head and heads of up to 128: the prompt kernel
PROMPTS = [(150, 150), (90, 70), (200, 129)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hs", [48, 64, 128])
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-16])
def test_prompts_of_zero_queries_and_keys(size, hs, half):
    """Rows of zeros (or hardly more) over keys of zeros: every visible position weighs the same. Keys whose scale is so
    small that its product with the row's is no float32, and ordinary ones, beside them."""
    c = Case(PROMPTS, 2, 1, hs, 16, half, seed=hs)
    c.q *= size
    for page in c.tables[0, :10]:
        c.kc[page], c.ks[page] = 0, 0
    c.ks[c.tables[1, :6]] = 1e-9
    got = c.run()
    assert np.isfinite(got).all()
    c.check(got)


@pytest.mark.parametrize("hs", [48, 64, 128])
@pytest.mark.parametrize("size", [1e-30, 1e25, 1e37])
def test_prompts_of_queries_of_any_size(size, hs):
    """float32 queries far outside float16's range, over keys that bring their scores back: scores stay as exact."""
    c = Case(PROMPTS, 2, 2, hs, 16, False, seed=8)
    c.q *= size
    c.ks *= np.float32(1 / size if size < 1e30 else 1e-37)
    c.check(c.run())


def test_store_of_the_smallest_scales():
    """float32 scales of one to seven of its smallest steps: the largest value may be up to 190 of them, and is stored as
    127, of its own sign."""
    step = 2.0 ** -149
    largest = np.array([64, 100, 127, 150, 190, 191, 260, 317, 318, 400, 700, 889])
    x = np.linspace(-1, 1, 32) * (largest * step)[:, None]
    (kc, ks), (vc, _) = store_case(x[:, None], -x[:, None], np.arange(12) * 16, 12, 16, 1, 32, False, 1)
    assert ks[4, 0] == np.float32(step) and (kc[4, 0, 0, [0, -1]] == [-127, 127]).all()
    for cache in (kc, vc):
        x32 = x.astype(np.float32).astype(np.float64) * (1 if cache is kc else -1)
        assert (np.sign(cache[:, 0, 0]) * np.sign(x32) >= 0).all()


def test_store_moves_the_smallest_scales():
    """A block whose scale goes from 1, 2, ... of float32's smallest steps to a few more: earlier integers that fall on a half
    go to the even one."""
    step = 2.0 ** -149
    n, hs = 9, 128
    x = np.tile(np.arange(128) - 64.0, (n, 1)) * step
    x[:, 0] = 127 * (1 + np.arange(n)) * step
    kv = store_case(x[:, None], -x[:, None], np.arange(n) * 16, n, 16, 1, hs, False, 1)
    y = np.zeros((n, hs))
    y[:, 0] = 127 * 6 * step * (1 + np.arange(n) // 3)
    store_case(y[:, None], -y[:, None], np.arange(n) * 16 + 1, n, 16, 1, hs, False, 1, kv=kv)


@pytest.mark.parametrize("starts,requests", [
    ([0, 5, 2, 7], [(50, 3), (50, 2), (50, 2)]), ([3, -4, 9, 1000], [(50, 3), (50, 2), (50, 2)]),
    ([0, 5, 3, 5], [(50, 3), (50, 2), (50, 2)]), ([0, 1, 2, 8], [(50, 3), (50, 2), (50, 2)]),
    ([-1, 2, 4, 6], [(900, 3), (50, 2), (50, 2)]), ([4, 4, 3, 3], [(900, 3), (50, 2), (50, 2)]),
    ([0, 100, 90, 300], [(200, 100), (150, 100), (700, 100)]), ([0, 100, 200, 301], [(200, 100), (150, 100), (700, 100)]),
    ([-2 ** 31, 100, 200, 300], [(200, 100), (150, 100), (700, 100)])])
@pytest.mark.parametrize("half", [False, True])
def test_attention_writes_nothing_where_starts_do_not_ascend(starts, requests, half):
    """starts that go down, begin below 0 or end behind the call's rows: no row is written, few rows and prompts, short
    tables and long ones."""
    c = Case(requests, 4, 2, 64, 16, half, seed=5)
    c.starts, c.behind = np.array(starts), 0
    c.upload()
    c.dq_wide = c.dq
    c.call()
    assert (host(c.out) == 7).all()


@pytest.mark.parametrize("at", [0, 127, 128, 640, 699])
def test_attention_finds_starts_that_do_not_ascend_among_many(at):
    """One pair of starts out of order among 700 requests, in any of the parts in which the kernels look them over."""
    c = Case([(30, 1)] * 699 + [(200, 150)], 4, 2, 64, 16, False, seed=6)
    c.behind = 0
    good = c.run()
    c.check(good)
    c.starts[at] = c.starts[at + 1] + 1 if at else -1
    c.upload()
    c.dq_wide = c.dq
    c.call()
    assert (host(c.out) == 7).all()


def test_attention_check_reads_the_scratch():
    """0 after a call, whatever the scratch held before it; the error that a kernel's wait would leave there (planted by the
    host here) as B200FWD_ETIMEOUT, until the next call."""
    lib = abi.load()
    c = Case([(200, 150), (90, 1)], 4, 2, 64, 16, False, seed=7)
    c.run()
    assert lib.b200k_cache8_attention_check(ptr(c.scratch), None) == 0
    c.scratch[1] = 104
    assert lib.b200k_cache8_attention_check(ptr(c.scratch), None) == abi.ETIMEOUT
    assert "104" in abi.last_error()
    c.call()
    assert lib.b200k_cache8_attention_check(ptr(c.scratch), None) == 0


# ------------------------------------------------------------------------------------------------------- precision

def exact(c):
    """(out, bound) of a case in float64. bound: what the header allows, by its terms, u = 2^-24 half a step of float32:
    - a query value is off by 2^-22 of itself (two float16 parts) or 2^-30 of its row's largest (digits of a byte);
    - a score's products, added in float32: (size / 8 + 4) times 4 u of the sum of their sizes (the tensor cores cut off);
    - the exponent: half a step of the score, the value scale's logarithm and the maximum each, twice, and 2^x;
    - sums over the positions: by steps of 64, 2 u each of the whole, and 64 u for joining the parts;
    - a weight in two float16 parts: 2^-22 of itself, and half a step, 2^-32, of the largest of its 64 positions (times value
      scale). Float16: half a step, 2^-11, and no finer than 2^-32 of the row's largest; the output half a step."""
    u = 2.0 ** -24
    size, group = c.hs, c.heads // c.nkv
    out, bound = np.zeros(c.q64.shape), np.zeros(c.q64.shape)
    for i, length in enumerate(c.lengths):
        rows, page = int(c.news[i]), c.tables[i, :-(-c.lengths[i] // c.block)].astype(int)
        for h in range(c.heads):
            kv = h // group
            k = (c.kc[page, kv].astype(np.float64) * c.ks[page, kv].astype(np.float64)[:, None, None]).reshape(-1, size)
            v_int = np.abs(c.vc[page, kv].astype(np.float64)).reshape(-1, size)
            vs = np.repeat(c.vs[page, kv].astype(np.float64), c.block)
            v = c.vc[page, kv].reshape(-1, size) * vs[:, None]
            for j in range(rows):
                t, seen = c.starts[i] + j, int(length) - rows + j + 1
                q = c.q64[t, h]
                s = k[:seen] @ q / np.sqrt(size)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ v[:seen]
                off = np.abs(k[:seen]) @ (np.abs(q) * 2.0 ** -22 + np.abs(q).max() * 2.0 ** -30)
                off += np.abs(k[:seen]) @ np.abs(q) * (size / 8 + 4) * 4 * u
                largest = np.abs(s).max() * 1.4427 + np.abs(np.log2(vs[:seen])).max()
                weight = (off / np.sqrt(size)).max() + (4 * largest + 64) * u + 2.0 ** -22
                whole = p @ np.abs(v[:seen])
                bound[t, h] = whole * (2 * weight + (2 * (seen // 64 + 1) + 64) * u)
                pv = p * vs[:seen]
                for at in range(0, seen, 64):
                    few = slice(at, min(seen, at + 64))
                    bound[t, h] += 2.0 ** -32 * (pv.max() if c.half else pv[few].max()) * v_int[few].sum(0)
                if c.half:
                    bound[t, h] += whole * 2.0 ** -11 + np.abs(out[t, h]) * 2.0 ** -11 + 2.0 ** -25
    return out, bound


def check_exact(c):
    got = c.run()
    want, bound = exact(c)
    off = np.abs(got - want)
    assert (off <= bound).all(), (np.argwhere(~(off <= bound))[:5], np.nanmax(off / bound), np.nanmax(off))
    return got


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("below", [9.0, 17.0, 22.0])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("requests,heads", [([(8192, 70)], 1), ([(20000, 1)] * 24, 1), ([(20000, 1)] * 12, 8)])
def test_attention_of_weights_far_below_the_largest(requests, heads, hs, below, half):
    """One position (of values 0) far above a flat rest, whose weights are what the output consists of."""
    c = Case(requests, heads, 1, hs, 64, half, seed=3)
    c.q[:] = 1
    c.kc[:], c.ks[:], c.vs[:] = 0, below / (127 * np.sqrt(hs)), 0.03
    c.vc[:] = np.abs(c.vc)
    for i in range(len(requests)):
        c.kc[c.tables[i, 0], :, 0] = 127
        c.vc[c.tables[i, 0], :, 0] = 0
    check_exact(c)


# ---------------------------------------------------------------------------------------------------- long prompts

@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hs", [64, 128])
def test_prompts_of_many_steps(hs, half):
    """Prompts of 25 and more steps of 64 positions, past the length of every ring of the prompt kernel: float32's maxima on
    their way from the softmax to the sums (8), scores (2 to 4), keys and values (4). Keys that grow along the first
    request, so that a row's maximum moves all the way; the same bits again."""
    c = Case([(1700, 1100), (1600, 1600), (2500, 70)], 2, 1, hs, 32, half, seed=hs)
    for j, b in enumerate(c.tables[0, :-(-1700 // 32)]):
        c.ks[b] = 0.0005 * (j + 1)
    got = check_exact(c)
    for _ in range(3):
        c.call()
        assert np.array_equal(c.result(), got)


# four, eight and sixteen rows a tile, and prompts
KINDS = [([(300, 1), (200, 1)], 4, 2), ([(300, 1), (200, 1)], 8, 2), ([(300, 3), (77, 2)], 8, 1), (PROMPTS, 2, 1)]


@pytest.mark.parametrize("half,outlier", [(False, 30), (False, 1000), (False, 1e5), (True, 30), (True, 1e4)])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("requests,heads,nkv", KINDS)
def test_attention_of_queries_with_an_outlier(requests, heads, nkv, hs, half, outlier):
    """A query value far above the others, where the keys are 0: the others' scores stay."""
    c = Case(requests, heads, nkv, hs, 16, half, seed=hs)
    c.q.reshape(c.n, heads, hs)[:, :, 5] = outlier
    c.kc[..., 5] = 0
    check_exact(c)


@pytest.mark.parametrize("requests,heads,nkv", KINDS)
def test_attention_of_the_largest_queries(requests, heads, nkv):
    """float32 queries up to the type's largest, over keys so small that the scores are ordinary."""
    c = Case(requests, heads, nkv, 64, 16, False, seed=9)
    c.q[:] = np.sign(c.q) * np.finfo(np.float32).max * np.random.default_rng(9).uniform(0.1, 1, c.q.shape)
    c.q[:, ::7] = np.finfo(np.float32).max * np.sign(c.q[:, ::7])
    c.ks[:] = 2.0 ** -133
    check_exact(c)


def test_attention_in_the_scratch_of_a_larger_call():
    """Fewer requests and tokens, but taller tiles, in a scratch sized for more of both: nothing behind it is touched."""
    lib, size = abi.load(), ctypes.c_uint64()
    c = Case([(3000, 3), (700, 2)], 8, 1, 64, 16, False, seed=2)
    c.upload()
    c.dq_wide = torch.cat([c.dq, c.dq[:1].expand(c.behind, -1)]).contiguous()
    abi.check(lib.b200k_cache8_attention_scratch(c.n + c.behind, 64, 8, 1, 64, 0, ctypes.byref(size)))
    room = int(size.value) // 4
    c.scratch = full(room + (1 << 20), -77, np.int32)
    c.call()
    c.check(c.result())
    assert (host(c.scratch)[room:] == -77).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hs", [16, 32, 80, 96])
def test_prompts_of_padded_heads(hs, half):
    """Head sizes that the prompt kernel pads to 64 or 128."""
    c = Case(PROMPTS, 3, 1, hs, 48, half, seed=hs)
    check_exact(c)


@pytest.mark.parametrize("half", [False, True])
def test_attention_of_single_tokens_in_wide_buffers(half):
    """A step of single tokens in buffers of 1000 rows, as a captured step makes it: the rows behind them stay."""
    c = Case([(300 + 17 * i, 1) for i in range(20)], 8, 2, 128, 32, half, seed=1)
    c.behind = 980
    check_exact(c)


@pytest.mark.parametrize("requests", [128, 129, 1000])
def test_attention_of_many_short_requests(requests):
    """Short tables of as many requests as one look takes, of one more, and of many."""
    rng = np.random.default_rng(requests)
    c = Case([(int(rng.integers(1, 80)), int(rng.integers(0, 2))) for _ in range(requests)], 4, 2, 32, 16, False, seed=requests)
    check_exact(c)


def test_attention_of_float16_gives_the_same_bits_again():
    c = Case([(20000, 1), (900, 1), (130, 3), (700, 200)], 8, 2, 128, 32, True, seed=12)
    first = c.run().copy()
    for _ in range(5):
        c.call()
        assert np.array_equal(c.result(), first)
