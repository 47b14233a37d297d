"""Where the paged 8-bit cache and its attention can go wrong: queries and keys of zeros, queries of any size, scales at
float32's lower end, starts that do not ascend, outliers among a query's values, weights far below the largest one, and
requests of more steps than the prompt kernel's rings hold. GPU only."""
import numpy as np
import pytest

from b200fwd import abi
from gpu_util import host, ptr
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
