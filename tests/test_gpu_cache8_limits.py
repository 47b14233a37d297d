"""Where the paged 8-bit cache and its attention can go wrong: queries and keys of zeros, queries of any size, scales at
float32's lower end, starts that do not ascend, outliers among a query's values, weights far below the largest one, and
requests of more steps than the prompt kernel's rings hold. GPU only."""
import numpy as np
import pytest

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
