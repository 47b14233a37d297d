"""b200k_logprobs against float64: log probabilities, entropy, the most probable ids (equal, ties by the lowest id), over
vocabularies from one logit to more than a cluster's registers hold, float32 and float16, masked and odd rows. GPU only."""
import numpy as np
import pytest

import cache8_plain as plain
from b200fwd import abi
from gpu_util import dev, full, host, ptr

pytestmark = pytest.mark.gpu


def run(x, targets, k, half, pad=0, offset=0, logprob=True, entropy=True):
    """x [rows][n] laid out with `pad` values between rows and `offset` values before the first"""
    lib = abi.load()
    rows, n = x.shape
    t = np.float16 if half else np.float32
    wide = np.full((rows, n + pad), 1e4, t)
    wide[:, :n] = x
    flat = dev(np.concatenate([np.full(offset, 1e4, t), wide.reshape(-1)]).view(np.uint16 if half else np.float32))
    out = [full(rows + 1, 3.0) for _ in range(2)] + [full((rows + 1, k), 3.0), full((rows + 1, k), 3, np.int32)]
    d = dev(np.asarray(targets, np.int32))
    abi.check(lib.b200k_logprobs(ptr(out[0]) if logprob else None, ptr(out[1]) if entropy else None,
                                 ptr(out[2]) if k else None, ptr(out[3]) if k else None,
                                 flat.data_ptr() + offset * (2 if half else 4), ptr(d), rows, n, n + pad, k, int(half), None))
    got = [host(o) for o in out]
    assert all((g[rows] == 3).all() for g in got)  # nothing behind the last row
    return [g[:rows] for g in got]


def check(got, x, targets, k):
    """A sum of exponentials: each off by 2^-22 (2^x) and by its argument's rounding, |d| 2^-23 of it, d e^d below 0.4; added
    in chains of up to 65 a round, three rounds, and 20 partial sums: 240 eps of the sum, eps = 2^-24. That is the error
    of log S; x - m is rounded once, and so is each of the two differences. The entropy is log S less a quotient of two
    such sums, the second one's terms up to the entropy's own size and the product's rounding."""
    eps = 2.0 ** -24
    chosen, entropy, top, ids = plain.logprobs(x, targets, k)
    assert np.array_equal(got[3], ids)
    for g, w in ((got[0], chosen), (got[2], top)):
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isneginf(g), np.isneginf(w))
        fine = np.isfinite(w)
        assert (np.abs(g[fine] - w[fine]) <= (240 + 3 * (np.abs(w[fine]) + 14)) * eps).all()
    assert np.array_equal(np.isnan(got[1]), np.isnan(entropy))
    fine = np.isfinite(entropy)
    assert (np.abs(got[1][fine] - entropy[fine]) <= (240 + 500 * entropy[fine] + 60) * eps).all()


def logits(rng, rows, n, half):
    x = rng.standard_normal((rows, n)) * 3
    x[:, :: 37] += 5
    return x.astype(np.float16 if half else np.float32)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,n,k,pad,offset", [
    (1, 1, 1, 0, 0), (3, 2, 2, 1, 1), (4, 7, 5, 0, 3), (2, 33, 32, 6, 2), (9, 320, 8, 0, 0), (5, 1000, 20, 3, 1),
    (1, 4097, 9, 0, 7), (200, 2049, 3, 0, 0), (5, 32000, 1, 0, 0), (3, 50257, 32, 0, 0), (2, 128256, 20, 0, 0),
    (150, 20011, 5, 0, 0), (1, 140001, 17, 2, 5), (2, 600001, 32, 0, 0)])
def test_logprobs_of_rows(rows, n, k, pad, offset, half):
    rng = np.random.default_rng(n)
    x = logits(rng, rows, n, half)
    targets = rng.integers(0, n, rows)
    check(run(x, targets, k, half, pad, offset), x, targets, k)


@pytest.mark.parametrize("half", [False, True])
def test_logprobs_of_masked_and_odd_rows(half):
    """Masks of -inf and of the lowest value, one token left, everything equal, rows without a distribution (all masked, an
    infinity, NaNs of either sign), targets that are no id or masked, zeros of both signs."""
    rng = np.random.default_rng(1)
    n, k = 5003, 12
    x = logits(rng, 14, n, half)
    low = np.finfo(x.dtype).min
    x[0, 100:] = -np.inf
    x[1, rng.permutation(n)[:4900]] = low
    x[2] = -np.inf
    x[2, 77] = 1.5                      # one token left: log probability 0, entropy 0
    x[3] = 0.25                         # all equal
    x[4] = low                          # all masked by the lowest value: all equal
    x[5] = -np.inf                      # nothing left
    x[6, 5000] = np.inf
    x[7, 3] = np.nan
    x[8, n - 1] = -np.nan
    x[9, :6] = -np.inf
    x[9, 6:] = np.where(np.arange(n - 6) % 2, 0.0, -0.0)
    x[10] = np.arange(n) % 5            # ties by the thousand
    x[11] = -np.inf
    x[11, [4000, 10, 4999]] = [1, 1, 2]  # fewer ids left than asked for: -inf, by the lowest id
    targets = rng.integers(0, n, 14)
    targets[0], targets[2], targets[11], targets[12], targets[13] = 4000, 77, 5, -1, n
    got = run(x, targets, k, half)
    check(got, x, targets, k)
    assert np.isneginf(got[0][0]) and got[0][2] == 0 and got[1][2] == 0
    for r in (5, 6, 7, 8):
        assert np.isnan(got[0][r]) and np.isnan(got[1][r]) and np.isnan(got[2][r]).all() and (got[3][r] == -1).all()


@pytest.mark.parametrize("n", [3000, 131073, 300007])
def test_logprobs_largest_in_one_thread(n):
    """The largest values so placed that few threads hold them all, and equal runs that fill the list."""
    rng = np.random.default_rng(n)
    x = logits(rng, 3, n, False)
    x[0, ::1024] += 50
    x[1, : 2000] = 40
    x[2, n - 600:] = 30
    targets = [0, 1999, n - 1]
    check(run(x, targets, 32, False), x, targets, 32)


def test_logprobs_parts_that_are_not_wanted():
    rng = np.random.default_rng(2)
    x = logits(rng, 4, 1000, False)
    targets = rng.integers(0, 1000, 4)
    whole = run(x, targets, 4, False)
    none = run(x, targets, 0, False)
    assert np.array_equal(none[0], whole[0]) and np.array_equal(none[1], whole[1])
    some = run(x, targets, 4, False, logprob=False, entropy=False)
    assert (some[0] == 3).all() and (some[1] == 3).all()
    assert np.array_equal(some[2], whole[2]) and np.array_equal(some[3], whole[3])


def test_logprobs_captured_and_replayed():
    import ctypes

    import torch

    lib = abi.load()
    rng = np.random.default_rng(3)
    rows, n, k = 6, 32000, 5
    x = dev(logits(rng, rows, n, False))
    targets = dev(rng.integers(0, n, rows).astype(np.int32))
    out = [full(rows, 0.0), full(rows, 0.0), full((rows, k), 0.0), full((rows, k), 0, np.int32)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        abi.check(lib.b200k_logprobs(*[ptr(o) for o in out], ptr(x), ptr(targets), rows, n, n, k, 0, stream))
    for _ in range(2):
        y = logits(rng, rows, n, False)
        x.copy_(torch.from_numpy(y))
        g.replay()
        check([host(o) for o in out], y, host(targets), k)
