"""The paged 8-bit cache on the GPU: block tables and store to the last integer, load and attention within what float32
arithmetic may be off (derived beside the float64 restatement in cache8_plain.py), the masks, pages, strides and shapes
where they can go wrong, and the whole run of a step as a server makes it. GPU only."""
import ctypes

import numpy as np
import pytest

import cache8_plain as plain
from b200fwd import abi
from gpu_util import dev, empty, full, host, ptr

pytestmark = pytest.mark.gpu


def i32(a):
    return dev(np.ascontiguousarray(a, np.int32))


def rows(a, half):
    """float rows as the device takes them (float16 bits or float32) and the numbers that they then are"""
    if half:
        h = np.ascontiguousarray(a, np.float16)
        return dev(h.view(np.uint16)), h.astype(np.float64)
    f = np.ascontiguousarray(a, np.float32)
    return dev(f), f.astype(np.float64)


def floats(t, half):
    return host(t).view(np.float16).astype(np.float64) if half else host(t).astype(np.float64)


# ---------------------------------------------------------------------------------------------------- block tables

class DeviceTables:
    def __init__(self, t):
        self.p = t
        self.tables, self.ring = i32(t.tables), i32(t.ring)
        self.state = i32([t.head, len(t.free), 0, 0])
        self.lengths = i32(t.lengths)

    def step(self, news, n, out_of_place=False, stream=None, with_rows=True):
        lib, t = abi.load(), self.p
        S = len(news)
        state, lengths = (empty(4, np.int32), empty(S, np.int32)) if out_of_place else (self.state, self.lengths)
        starts, slots, seq, pos = (full(x, -5, np.int32) for x in (S + 1, n + 1, n + 1, n + 1))
        d = i32(news)
        abi.check(lib.b200k_block_tables(ptr(self.tables), ptr(self.ring), ptr(state), ptr(lengths), ptr(starts), ptr(slots),
                                         ptr(seq) if with_rows else None, ptr(pos) if with_rows else None, ptr(self.state),
                                         ptr(self.lengths), ptr(d), S, t.width, t.blocks, t.block, n, stream))
        got = [host(x) for x in (starts, slots, seq, pos, state, lengths)]
        self.state, self.lengths = state, lengths
        return got


def same_step(d, news, n, **how):
    t = d.p
    want = t.step(news, n)
    starts, slots, seq, pos, state, lengths = d.step(news, n, **how)
    assert state[2] == want[0]
    assert np.array_equal(starts, want[1])
    for g, w in zip((slots, seq, pos), want[2:]):
        if how.get("with_rows", True) or g is slots:
            assert np.array_equal(g[:n], w)
        assert g[n] == -5  # nothing behind the step's rows
    assert np.array_equal(lengths, t.lengths)
    assert state[0] == t.head and state[1] == len(t.free) and state[3] == want[1][-1]
    assert np.array_equal(host(d.tables), t.tables)
    assert np.array_equal(host(d.ring), t.ring)
    return want[0]


@pytest.mark.parametrize("S,width,block,most,seed", [
    (1, 4, 16, 40, 0), (3, 9, 32, 100, 1), (64, 30, 16, 60, 2), (511, 12, 48, 90, 3), (513, 12, 16, 50, 4),
    (1500, 7, 64, 100, 5), (70, 300, 256, 9000, 6)])
def test_block_tables_follow_the_requests(S, width, block, most, seed):
    """Prompts, single tokens, tokens taken back and finished requests over several steps, in place and not, with the
    ring turning over; one thread block's sizes and the cluster's."""
    rng = np.random.default_rng(seed)
    blocks = S * width * 2 // 3 + width
    d = DeviceTables(plain.Tables(S, width, blocks, block, blocks - 3, rng.permutation(blocks)))
    granted = 0
    for step in range(8):
        kind = rng.random(S)
        news = np.where(kind < 0.3, rng.integers(0, most + 1, S), np.where(kind < 0.7, 1, 0))
        news = np.where(kind > 0.85, -rng.integers(0, most + 1, S), news)
        news = np.where(kind > 0.95, -2 ** 31, news)
        news = np.minimum(news, width * block - d.p.lengths)  # (the width's refusal has a test of its own)
        total = int(np.maximum(news, 0).sum())
        granted += same_step(d, news, total + int(rng.integers(0, 9)), out_of_place=step % 2 == 1, with_rows=step != 3) == 0
    assert granted >= 2


@pytest.mark.parametrize("n", [4095, 4096, 4097, 5000, 9001])
def test_block_tables_of_many_rows(n):
    """Steps around the rows from which another kernel writes them: requests without tokens among long ones and at both
    ends, a request that ends a step's rows, steps that are not granted, blocks' ends between two warps' rows."""
    rng = np.random.default_rng(n)
    d = DeviceTables(plain.Tables(9, 700, 700, 16, 690, rng.permutation(700)))
    assert same_step(d, [0, 0, 1500, 1, 0, n - 1503, 0, 2, 0], n) == 0
    assert same_step(d, [3, -1500, 0, 1, 0, 11200, 0, 0, 0], n) == abi.TABLES_WIDTH
    assert same_step(d, [3, -1500, 0, 1, 0, 0, 0, n, 0], n) == abi.TABLES_TOKENS
    assert same_step(d, [1, -2 ** 31, -2 ** 31, 0, 0, -2 ** 31, 129, 127, 0], n, with_rows=False) == 0
    assert same_step(d, [0, 128, 0, 0, 1, 0, 0, 0, 4000], n, out_of_place=True) == (0 if n >= 4129 else abi.TABLES_TOKENS)


def test_block_tables_grant_all_or_nothing():
    d = DeviceTables(plain.Tables(3, 4, 6, 16, 2, [5, 1, 3, 0, 2, 4]))
    assert same_step(d, [17, 16, 1], 34) == 0                      # four of six blocks
    assert same_step(d, [16, 17, 16], 60) == abi.TABLES_BLOCKS     # five more
    assert same_step(d, [1, 1, 1], 2) == abi.TABLES_TOKENS
    assert same_step(d, [48, -16, 0], 60) == abi.TABLES_WIDTH      # 65 positions of 64
    assert same_step(d, [0, -16, -1], 0) == 0                      # two blocks come back, no tokens
    assert same_step(d, [47, 0, 0], 47) == 0                       # exactly the table row's width
    assert same_step(d, [-64, 32, 32], 64) == abi.TABLES_BLOCKS    # given back in this step: not taken in it
    assert same_step(d, [-64, 0, 0], 0) == 0
    assert same_step(d, [0, 64, 32], 96) == 0


@pytest.mark.parametrize("state,lengths", [([-1, 3, 0, 0], [4, 4]), ([6, 3, 0, 0], [4, 4]), ([0, 7, 0, 0], [4, 4]),
                                           ([0, -1, 0, 0], [4, 4]), ([0, 3, 0, 0], [-1, 4]), ([0, 3, 0, 0], [4, 65]),
                                           ([0, 6, 0, 0], [64, 4])])
def test_block_tables_refuse_what_cannot_be(state, lengths):
    """A head or count outside the ring, a length below 0 or past its row, more blocks given back than the ring has room
    for: the status says so and nothing moves."""
    t = plain.Tables(2, 4, 6, 16, 0, [])
    d = DeviceTables(t)
    d.state, d.lengths = i32(state), i32(lengths)
    d.tables = full((2, 4), 1, np.int32)
    starts, slots, seq, pos, after, still = d.step([-64, 1], 5)
    assert list(after) == [state[0], state[1], abi.TABLES_INPUT, 0]
    assert list(still) == lengths and not starts.any()
    assert (slots[:5] == -1).all() and (seq[:5] == -1).all() and (pos[:5] == -1).all()
    assert (host(d.tables) == 1).all() and (host(d.ring) == -9).all()


def test_block_tables_pass_on_no_bad_id():
    """An id in the ring or the table that is no block: its tokens have slot -1."""
    t = plain.Tables(2, 4, 6, 16, 0, [2, 3, 4])
    d = DeviceTables(t)
    d.ring = i32([2, 99, -4, 0, 0, 0])
    starts, slots, _, pos, state, _ = d.step([16, 20], 36)
    assert state[2] == 0
    assert np.array_equal(slots[:16], 32 + np.arange(16)) and (slots[16:36] == -1).all()
    assert np.array_equal(pos[16:36], np.arange(20))


# ----------------------------------------------------------------------------------------------------- store, load

def pool(rng, blocks, nkv, block, hs):
    """a pool as it might stand: every byte and scale something"""
    return (rng.integers(-127, 128, (blocks, nkv, block, hs)).astype(np.int8),
            np.exp(rng.standard_normal((blocks, nkv))).astype(np.float32) * np.float32(0.05))


def store_case(k, v, slots, blocks, block, nkv, hs, half, seed, pad=0, kv=None):
    """store's caches against the restatement's, to the last integer and scale"""
    rng = np.random.default_rng(seed)
    (kc, ks), (vc, vs) = kv or (pool(rng, blocks, nkv, block, hs), pool(rng, blocks, nkv, block, hs))
    n, row = len(slots), nkv * hs
    wide = lambda x: np.concatenate([x.reshape(n, row), np.full((n, pad), 1e4)], 1)  # noqa: E731
    dk, k64 = rows(wide(k), half)
    dv, v64 = rows(wide(v), half)
    d = [dev(x) for x in (kc, ks, vc, vs)]
    ds = i32(slots)
    abi.check(abi.load().b200k_cache8_store(*[ptr(x) for x in d], ptr(dk), ptr(dv), ptr(ds), n, row + pad, row + pad, blocks,
                                            block, nkv, hs, int(half), None))
    kc, ks, vc, vs = (x.copy() for x in (kc, ks, vc, vs))
    plain.store(kc, ks, k64[:, :row].reshape(n, nkv, hs), slots, block)
    plain.store(vc, vs, v64[:, :row].reshape(n, nkv, hs), slots, block)
    for got, want in zip(d, (kc, ks, vc, vs)):
        got = host(got)
        assert np.array_equal(got, want, equal_nan=got.dtype == np.float32), np.argwhere(got != want)[:5]
    return (kc, ks), (vc, vs)


SHAPES = [(1, 16, 16), (2, 48, 16), (1, 144, 32), (8, 128, 32), (3, 64, 64), (2, 80, 48), (1, 256, 256), (5, 96, 16), (4, 112, 128)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nkv,hs,block", SHAPES)
def test_store_quantizes_blocks(nkv, hs, block, half):
    """Prompts over whole and part blocks, single tokens into begun blocks (scales that grow, and that stay), rows without
    a slot among them, rows with a stride: integers and scales equal the definition's."""
    rng = np.random.default_rng(nkv * 1000 + hs + block)
    order = rng.permutation(24)
    slots = []
    at = lambda b, lo, hi: list(order[b] * block + np.arange(lo, hi))  # noqa: E731
    slots += at(0, 0, block) + at(1, 0, block) + at(2, 0, 5)      # a prompt of two blocks and a bit
    slots += at(3, 7, block) + at(4, 0, 1)                        # a request that goes on, to a new block
    slots += at(5, block - 1, block) + [-1, 24 * block, 2 ** 31 - 1, -2 ** 31] + at(6, 3, 4) + at(7, 0, 1) + [-1]
    slots += at(8, 1, 2) + at(9, block // 2, block // 2 + 3)
    n = len(slots)
    loud = np.exp(rng.standard_normal((n, nkv, 1)))
    make = lambda: rng.standard_normal((n, nkv, hs)) * loud * 2  # noqa: E731
    store_case(make(), make(), np.array(slots), 24, block, nkv, hs, half, 7, pad=16)


@pytest.mark.parametrize("n", [1, 3, 257, 2100])
def test_store_of_single_tokens(n):
    """One token a request, as a decode step stores them (each way that the kernel divides a call's rows)."""
    rng = np.random.default_rng(n)
    blocks, block = n + 3, 16
    slots = rng.permutation(blocks)[:n] * block + rng.integers(0, block, n)
    make = lambda: rng.standard_normal((n, 1, 32)) * np.exp(2 * rng.standard_normal((n, 1, 1)))  # noqa: E731
    store_case(make(), make(), slots, blocks, block, 1, 32, False, n)


def test_store_token_by_token():
    """A block filled one token at a time, each louder or softer than the last: its scale never falls, its earlier integers
    follow every time it grows, and beginning it anew forgets them."""
    rng = np.random.default_rng(5)
    kv = None
    for t in list(range(16)) + [0, 1]:
        x = rng.standard_normal((1, 2, 64)) * 2.0 ** rng.integers(-3, 4)
        kv = store_case(x, -x, np.array([3 * 16 + t]), 6, 16, 2, 64, False, 11, kv=kv)


@pytest.mark.parametrize("half", [False, True])
def test_store_of_odd_values(half):
    """Zeros; the type's largest and smallest; values just off and on a half step; a lone value; NaN and infinities, in the
    call and in a begun block."""
    rng = np.random.default_rng(3)
    block, hs = 16, 32
    big, tiny = (65504.0, 6e-8) if half else (3.4e38, 1.4e-45)
    x = np.zeros((10, 1, hs))
    x[1] = big * rng.uniform(-1, 1, (1, hs))
    x[2] = tiny * rng.integers(-3, 4, (1, hs))
    x[3, 0, :] = (np.arange(hs) + 0.5) / 2           # scale 1/8 exactly: halves on the step's grid
    x[3, 0, 0] = 127 / 8
    x[4, 0, :] = np.float32(0.1) * (np.arange(hs) + 0.5)
    x[4, 0, 0] = np.float32(12.7)
    x[5, 0, 3] = -4.0
    x[6, 0, 1], x[7, 0, 2], x[8, 0, 3] = np.nan, np.inf, -np.inf
    x[9] = rng.standard_normal((1, hs))
    slots = np.arange(10) * block
    (kc, ks), _ = kv = store_case(x, x[::-1], slots, 11, block, 1, hs, half, 1)
    assert ks[0, 0] == 0 and np.isnan(ks[6:9, 0]).all() and not kc[6:9, 0, 0].any()
    # the next token of each block: a block with NaN stays so, zeros and tiny ones come to the new scale
    store_case(x[::-1], x, slots + 1, 11, block, 1, hs, half, 2, kv=kv)


def test_store_scales_below_an_inverse():
    """float32 blocks whose scale has no float32 inverse."""
    rng = np.random.default_rng(8)
    x = np.array([1e-37, 1e-36, 1.27e-35, 3e-39, 2e-43, 9e-38]).reshape(6, 1, 1) * rng.uniform(-1, 1, (6, 1, 16))
    store_case(x, x, np.arange(6) * 16, 6, 16, 1, 16, False, 4)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nkv,hs,block", SHAPES)
def test_load_gives_the_stored_values(nkv, hs, block, half):
    """q s in float32 (rounded once more to float16): to the bit, in any order of slots, the same slot twice; rows without
    a slot stay."""
    rng = np.random.default_rng(hs)
    blocks, n, pad = 9, 37, 8
    kc, ks = pool(rng, blocks, nkv, block, hs)
    vc, vs = pool(rng, blocks, nkv, block, hs)
    slots = rng.integers(0, blocks * block, n)
    slots[[3, 17]] = slots[5]
    slots[[8, 9, 36]] = [-1, blocks * block, -2 ** 31]
    row = nkv * hs
    k, v = (full((n, row + pad), 7, np.uint16 if half else np.float32) for _ in range(2))
    d = [dev(x) for x in (kc, ks, vc, vs)]
    ds = i32(slots)
    abi.check(abi.load().b200k_cache8_load(ptr(k), ptr(v), *[ptr(x) for x in d], ptr(ds), n, row + pad, row + pad, blocks,
                                           block, nkv, hs, int(half), None))
    for got, cache, scales in ((k, kc, ks), (v, vc, vs)):
        got = host(got, np.uint16 if half else np.uint32)
        want = np.full((n, row + pad), 7, np.float32).view(np.uint32) if not half else np.full((n, row + pad), 7, np.uint16)
        for i, s in enumerate(slots):
            if 0 <= s < blocks * block:
                x = cache[s // block, :, s % block].astype(np.float32) * scales[s // block][:, None]
                x = x.reshape(-1)
                want[i, :row] = x.astype(np.float16).view(np.uint16) if half else x.view(np.uint32)
        assert np.array_equal(got, want)


# ------------------------------------------------------------------------------------------------------- attention

class Case:
    """A pool, tables and queries of requests given as (positions, new tokens)."""

    def __init__(self, requests, heads, nkv, hs, block, half, seed=0, width=None, q_size=1.5):
        rng = np.random.default_rng(seed)
        self.heads, self.nkv, self.hs, self.block, self.half = heads, nkv, hs, block, half
        self.lengths = np.array([r[0] for r in requests], np.int64)
        self.news = np.array([r[1] for r in requests], np.int64)
        self.starts = np.concatenate([[0], np.cumsum(self.news)])
        self.n = int(self.starts[-1])
        need = -(-self.lengths // block)
        self.width = width or max(1, int(need.max()))
        self.blocks = int(need.sum()) + 3
        order = rng.permutation(self.blocks)
        self.tables = rng.integers(-2 ** 31, 2 ** 31 - 1, (len(requests), self.width))  # what no row sees is anything
        at = 0
        for i, m in enumerate(need):
            self.tables[i, :m] = order[at:at + m]
            at += m
        self.kc, self.ks = pool(rng, self.blocks, nkv, block, hs)
        self.vc, self.vs = pool(rng, self.blocks, nkv, block, hs)
        self.ks /= 4
        self.q = rng.standard_normal((self.n, heads * hs)) * q_size
        self.q_pad, self.out_pad, self.behind = 0, 0, 2

    def upload(self):
        q = np.concatenate([self.q, np.full((self.n, self.q_pad), np.nan)], 1)
        self.dq, q64 = rows(q, self.half)
        self.q64 = q64[:, :self.heads * self.hs].reshape(self.n, self.heads, self.hs)
        self.dev = [dev(x) for x in (self.kc, self.ks, self.vc, self.vs)]
        self.dt, self.ds, self.dl = i32(self.tables), i32(self.starts), i32(self.lengths)
        self.out = full((self.n + self.behind, self.heads * self.hs + self.out_pad), 7, np.uint16 if self.half else np.float32)
        size = ctypes.c_uint64()
        abi.check(abi.load().b200k_cache8_attention_scratch(self.n + self.behind, len(self.lengths), self.heads, self.nkv,
                                                            self.hs, int(self.half), ctypes.byref(size)))
        self.scratch = empty(int(size.value) // 4, np.int32)
        self.scratch.fill_(-1)  # (NaNs, and indices that would be out of range)

    def call(self, stream=None):
        """rows behind the last request are in the call, and belong to none"""
        row = self.heads * self.hs
        abi.check(abi.load().b200k_cache8_attention(
            ptr(self.out), ptr(self.dq_wide), *[ptr(x) for x in self.dev], ptr(self.dt), ptr(self.ds), ptr(self.dl),
            self.n + self.behind, len(self.lengths), self.width, self.blocks, self.block, self.heads, self.nkv, self.hs,
            row + self.q_pad, row + self.out_pad, int(self.half), ptr(self.scratch), stream))

    def run(self):
        import torch

        self.upload()
        self.dq_wide = torch.cat([self.dq, self.dq[:1].expand(self.behind, -1)]) if self.behind else self.dq
        self.dq_wide = self.dq_wide.contiguous()
        self.call()
        return self.result()

    def result(self):
        got = host(self.out)
        keep = got[self.n:].reshape(-1), got[:, self.heads * self.hs:].reshape(-1)
        assert all((x == 7).all() for x in keep)  # rows behind the last request, and between the rows
        got = got[:self.n, :self.heads * self.hs]
        got = np.ascontiguousarray(got).view(np.float16) if self.half else got
        return got.astype(np.float64).reshape(self.n, self.heads, self.hs)

    def check(self, got):
        want, bound = plain.attention(self.q64, self.kc, self.ks, self.vc, self.vs, self.tables, self.starts, self.lengths,
                                      self.block, self.heads // self.nkv, self.half)
        off = np.abs(got - want)
        assert (off <= bound).all(), (np.argwhere(~(off <= bound))[:5], np.nanmax(off / bound))


# (positions, new tokens) of the requests; heads, kv heads, head size, block
ATTENTION = [
    ([(1, 1)], 1, 1, 16, 16),
    ([(17, 1), (16, 1), (15, 1), (33, 1)], 4, 2, 64, 16),
    ([(200, 1), (1, 1), (64, 1), (5, 0), (333, 1)], 8, 2, 128, 32),
    ([(0, 0), (40, 1), (0, 0), (0, 0), (97, 1), (0, 0)], 6, 6, 48, 48),
    ([(70, 3), (2, 2), (300, 5)], 7, 1, 80, 16),
    ([(129, 1), (500, 1)], 32, 8, 128, 64),
    ([(129, 9), (40, 40)], 6, 2, 96, 32),
    ([(257, 2)], 71, 1, 64, 16),
    ([(511, 1), (600, 2)], 4, 4, 192, 256),
    ([(100, 1), (77, 3)], 16, 2, 256, 16),
    ([(3000, 1)], 4, 1, 128, 16),
    ([(5001, 1), (2, 1), (17, 1)], 8, 8, 64, 128),
    ([(260, 260), (100, 37)], 8, 2, 64, 32),
    ([(300, 300), (77, 1), (190, 129)], 16, 4, 128, 64),
    ([(450, 200), (128, 128), (31, 31)], 3, 1, 112, 16),
    ([(700, 140)], 24, 2, 256, 32),
    ([(3, 5), (0, 2), (1, 1), (0, 1), (18, 20)], 4, 2, 32, 16),   # fewer positions than tokens: rows that see nothing
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("requests,heads,nkv,hs,block", ATTENTION)
def test_attention_of_requests(requests, heads, nkv, hs, block, half):
    c = Case(requests, heads, nkv, hs, block, half, seed=heads + hs)
    got = c.run()
    c.check(got)
    for i, (length, fresh) in enumerate(requests):
        for j in range(max(0, fresh - length)):
            assert not got[c.starts[i] + j].any()  # a row that sees no position is 0


@pytest.mark.parametrize("half", [False, True])
def test_attention_many_requests(half):
    """More requests than a thread block has threads, most of them short, some with nothing to do."""
    rng = np.random.default_rng(9)
    requests = [(int(rng.integers(1, 60)), int(rng.integers(0, 3))) for _ in range(300)]
    requests = [(max(l, c), c) for l, c in requests]
    requests[150] = (2500, 1)
    c = Case(requests, 4, 2, 64, 16, half, seed=4)
    c.check(c.run())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("requests", [[(90, 1), (300, 1)], [(150, 150), (60, 7)]])
def test_attention_strides(requests, half):
    """Queries within wider rows (a fused q|k|v buffer) and outputs with room between them."""
    c = Case(requests, 4, 2, 64, 16, half, seed=1)
    c.q_pad, c.out_pad = 264, 16
    c.check(c.run())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("fresh", [1, 150])
def test_attention_bad_pages(fresh, half):
    """Table entries that are no block: NaN in the rows that see one of their positions, no other row moved."""
    c = Case([(200, fresh), (200, fresh), (190, fresh)], 4, 2, 64, 16, half, seed=2)
    c.tables[1, 12] = c.blocks      # positions 192 .. 199
    c.tables[2, 0] = -1
    got = c.run()
    good = c.tables.copy()
    good[1, 12], good[2, 0] = 0, 0
    c.tables = good
    blind = np.zeros(c.n, bool)
    blind[c.starts[1] + max(0, fresh - 8):c.starts[2]] = True
    blind[c.starts[2]:] = True
    assert np.isnan(got[blind]).all()
    want, bound = plain.attention(c.q64, c.kc, c.ks, c.vc, c.vs, c.tables, c.starts, c.lengths, c.block, 2, half)
    assert (np.abs(got - want) <= bound)[~blind].all()


@pytest.mark.parametrize("fresh", [1, 40, 200])
def test_attention_past_the_table(fresh):
    """More positions than the table row has room for: NaN where a row sees one of them."""
    c = Case([(200, fresh)], 2, 1, 64, 16, False, seed=3)
    c.lengths[0] = 13 * 16 + 5  # the row has 13 blocks
    got = c.run()
    blind = np.arange(c.n) >= c.n - 5
    assert np.isnan(got[blind]).all() and not np.isnan(got[~blind]).any()


@pytest.mark.parametrize("starts,lengths", [([0, 5, 2, 7], [50, 50, 50]), ([3, -4, 9, 1000], [50, 50, 50]),
                                            ([0, 1, 2, 3], [-5, 2 ** 31 - 1, 50]), ([2 ** 31 - 1, -2 ** 31, 0, 7], [1, 1, 1])])
def test_attention_of_inconsistent_requests(starts, lengths):
    """starts that do not ascend within the rows, lengths that cannot be: in bounds, and it ends."""
    c = Case([(50, 3), (50, 2), (50, 2)], 4, 2, 64, 16, False, seed=5)
    c.tables[:] = np.clip(c.tables, 0, c.blocks - 1)
    c.starts, c.lengths = np.array(starts), np.array(lengths)
    c.behind = 0
    c.run_unchecked = True
    c.upload()
    c.dq_wide = c.dq
    c.call()
    host(c.out)


def test_attention_masked_blocks_may_hold_anything():
    """The block that a request's last position is in: what stands behind that position does not count, nor do the scales
    of blocks that no row sees."""
    c = Case([(37, 1), (20, 12)], 4, 2, 64, 16, False, seed=6, width=5)
    seen = set(c.tables[0, :3]) | set(c.tables[1, :2])
    others = [b for b in range(c.blocks) if b not in seen]
    c.tables[:, 3:] = others[0]
    c.ks[others], c.vs[others] = np.nan, np.inf
    want = c.run()
    c.check(want)
    for b, behind in ((c.tables[0, 2], 5), (c.tables[1, 1], 4)):
        c.kc[b, :, behind:] = -127
        c.vc[b, :, behind:] = 127
    assert np.array_equal(c.run(), want)


def test_attention_of_scales_far_apart():
    """Blocks of zeros (scale 0), value scales from 1e-20 to 1e10, key scales of 0, NaN scales in what a row sees."""
    c = Case([(96, 1), (96, 50), (16, 1), (48, 1)], 2, 1, 64, 16, False, seed=7)
    t = c.tables
    c.vs[t[0, 0]], c.vc[t[0, 0]] = 0, 0
    c.vs[t[0, 1]], c.vs[t[0, 2]] = 1e-20, 1e10
    c.ks[t[1, 0]], c.kc[t[1, 0]] = 0, 0
    c.vs[t[1, 3]] = 0
    c.vc[t[1, 3]] = 0
    c.vs[t[2, 0]], c.vc[t[2, 0]] = 0, 0          # a request whose every value is 0
    c.check(c.run())
    c.ks[t[3, 1]] = np.nan
    assert np.isnan(c.run()[c.starts[3]:]).all()
    c.ks[t[3, 1]], c.vs[t[3, 2]] = 0.1, np.nan
    assert np.isnan(c.run()[c.starts[3]:]).all()


@pytest.mark.parametrize("size", [1e-30, 1e25, 1e37])
def test_attention_of_queries_of_any_size(size):
    """float32 queries far outside float16's range: scores stay as exact (the softmax flat, or one-hot)."""
    c = Case([(50, 1), (60, 20)], 2, 2, 48, 16, False, seed=8)
    c.q *= size
    c.ks *= np.float32(1 / size if size < 1e30 else 1e-37)
    c.check(c.run())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hs", [48, 128])
def test_attention_of_queries_that_are_no_numbers(hs, half):
    """A query with an infinity or a NaN in it gives NaN, and changes no other row or head. (The keys of the first block
    are such that an infinity's scores are all -inf there.)"""
    c = Case([(50, 1), (60, 20), (150, 100), (100, 100)], 4, 2, hs, 16, half, seed=11)
    c.kc[c.tables[3, 0], :, :, 1] = -np.abs(c.kc[c.tables[3, 0], :, :, 1]) - 1
    want = c.run()
    c.check(want)
    odd = [(0, 1, np.nan), (5, 0, np.inf), (20, 3, -np.inf), (21, 2, np.nan), (77, 1, np.inf), (120, 3, -np.inf),
           (121, 0, np.inf), (125, 2, np.inf), (200, 3, np.nan)]
    is_odd = np.zeros((c.n, c.heads), bool)
    for row, head, x in odd:
        c.q[row, head * hs + 1] = x
        is_odd[row, head] = True
    got = c.run()
    assert np.isnan(got[is_odd]).all(), np.argwhere(~np.isnan(got).any(2) & is_odd)
    assert np.array_equal(got[~is_odd], want[~is_odd])


def test_attention_sharp_and_growing_scores():
    """The running maximum moves at every unit, up to scores in the hundreds."""
    c = Case([(400, 1), (300, 30)], 4, 2, 64, 16, False, seed=10)
    c.q[:] = np.abs(c.q) * 3
    for i in range(2):
        for j, b in enumerate(c.tables[i, :-(-c.lengths[i] // 16)]):
            c.kc[b] = np.abs(c.kc[b])
            c.ks[b] = 0.002 * (j + 1)
    c.check(c.run())


def test_attention_gives_the_same_bits_again():
    c = Case([(2000, 1), (900, 1), (130, 3)], 8, 2, 128, 32, False, seed=12)
    first = c.run().copy()
    for _ in range(3):
        c.call()
        assert np.array_equal(c.result(), first)


def test_attention_offsets_past_32_bits():
    """A pool of more than 2^32 bytes a side, the request's blocks at its end."""
    import torch

    nkv, hs, block, blocks = 4, 256, 256, 17000  # 4.4 GB a side
    c = Case([(700, 1), (513, 200)], 8, nkv, hs, block, True, seed=13)
    c.upload()
    c.dq_wide = torch.cat([c.dq, c.dq[:1].expand(c.behind, -1)]).contiguous()
    small, caches = c.blocks, []
    for x in c.dev:
        wide = torch.zeros((blocks, *x.shape[1:]), dtype=x.dtype, device="cuda")
        wide[blocks - small:] = x
        caches.append(wide)
    c.dev, held = caches, c.dev
    c.dt = i32(np.where((c.tables >= 0) & (c.tables < small), c.tables + blocks - small, -1))
    c.blocks = blocks
    c.call()
    c.check(c.result())
    # load and store there too
    lib, slot = abi.load(), (blocks - 1) * block + 255
    x = torch.randn(1, nkv * hs, device="cuda")
    k, v = torch.empty_like(x), torch.empty_like(x)
    d = i32([(blocks - 1) * block])
    p = [ptr(t) for t in caches]
    abi.check(lib.b200k_cache8_store(*p, ptr(x), ptr(x), ptr(d), 1, nkv * hs, nkv * hs, blocks, block, nkv, hs, 0, None))
    abi.check(lib.b200k_cache8_load(ptr(k), ptr(v), *p, ptr(d), 1, nkv * hs, nkv * hs, blocks, block, nkv, hs, 0, None))
    step = x.view(nkv, hs).abs().amax(1, keepdim=True) / 127
    assert slot < 2 ** 31 and (k.view(nkv, hs) - x.view(nkv, hs)).abs().le(step * 0.5001).all() and torch.equal(k, v)


# --------------------------------------------------------------------------------------------------- a server's run

class Server:
    """A pool with its requests as a program keeps them, each step: tables, store, attention."""

    def __init__(self, S, heads, nkv, hs, block, width, half, n):
        rng = np.random.default_rng(21)
        self.S, self.heads, self.nkv, self.hs, self.block, self.width, self.half, self.n = S, heads, nkv, hs, block, width, half, n
        self.blocks = S * width
        self.tables, self.ring = full((S, width), 0, np.int32), i32(rng.permutation(self.blocks))
        self.state, self.lengths, self.news = i32([0, self.blocks, 0, 0]), full(S, 0, np.int32), full(S, 0, np.int32)
        self.starts, self.slots, self.seq, self.pos = (empty(x, np.int32) for x in (S + 1, n, n, n))
        self.kc, self.vc = (full((self.blocks, nkv, block, hs), 99, np.int8) for _ in range(2))
        self.ks, self.vs = (full((self.blocks, nkv), np.nan, np.float32) for _ in range(2))
        t = np.uint16 if half else np.float32
        self.q, self.out = full((n, heads * hs), 0, t), full((n, heads * hs), 0, t)
        self.k, self.v = full((n, nkv * hs), 0, t), full((n, nkv * hs), 0, t)
        size = ctypes.c_uint64()
        abi.check(abi.load().b200k_cache8_attention_scratch(n, S, heads, nkv, hs, int(half), ctypes.byref(size)))
        self.scratch = empty(int(size.value) // 4, np.int32)

    def step(self, stream=None):
        lib, p = abi.load(), ptr
        pool_ = p(self.kc), p(self.ks), p(self.vc), p(self.vs)
        row = self.nkv * self.hs
        abi.check(lib.b200k_block_tables(p(self.tables), p(self.ring), p(self.state), p(self.lengths), p(self.starts),
                                         p(self.slots), p(self.seq), p(self.pos), p(self.state), p(self.lengths), p(self.news),
                                         self.S, self.width, self.blocks, self.block, self.n, stream))
        abi.check(lib.b200k_cache8_store(*pool_, p(self.k), p(self.v), p(self.slots), self.n, row, row, self.blocks, self.block,
                                         self.nkv, self.hs, int(self.half), stream))
        row = self.heads * self.hs
        abi.check(lib.b200k_cache8_attention(p(self.out), p(self.q), *pool_, p(self.tables), p(self.starts), p(self.lengths),
                                             self.n, self.S, self.width, self.blocks, self.block, self.heads, self.nkv, self.hs,
                                             row, row, int(self.half), p(self.scratch), stream))

    def fill(self, rng, news):
        """this step's inputs, written into the step's buffers"""
        import torch

        self.news.copy_(torch.tensor(list(news), dtype=torch.int32))
        t = torch.float16 if self.half else torch.float32
        for x in (self.q, self.k, self.v):
            y = torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32) * 1.5).to(t)
            x.copy_(y.view(torch.int16) if self.half else y)

    def check(self, twin, before, news):
        """against the restatement's tables, store and attention (twin: tables and caches that it keeps)"""
        t, kc, ks, vc, vs = twin
        status, starts, slots, _, _ = t.step(news, self.n)
        assert status == 0 and host(self.state)[2] == 0
        assert np.array_equal(host(self.starts), starts) and np.array_equal(host(self.slots), slots)
        k, v, q = (floats(x, self.half) for x in (self.k, self.v, self.q))
        plain.store(kc, ks, k.reshape(self.n, self.nkv, self.hs), slots, self.block)
        plain.store(vc, vs, v.reshape(self.n, self.nkv, self.hs), slots, self.block)
        for got, want in ((self.kc, kc), (self.ks, ks), (self.vc, vc), (self.vs, vs)):
            assert np.array_equal(host(got), want, equal_nan=want.dtype == np.float32)
        want, bound = plain.attention(q.reshape(self.n, self.heads, self.hs), kc, ks, vc, vs, t.tables, starts, t.lengths,
                                      self.block, self.heads // self.nkv, self.half)
        got = floats(self.out, self.half).reshape(self.n, self.heads, self.hs)
        live = slice(0, int(starts[-1]))
        assert (np.abs(got[live] - want[live]) <= bound[live]).all()
        assert np.array_equal(got[live.stop:], before[live.stop:])


def twin_of(s):
    t = plain.Tables(s.S, s.width, s.blocks, s.block, 0, host(s.ring).tolist())
    t.tables[:] = 0
    return t, host(s.kc).copy(), host(s.ks).copy(), host(s.vc).copy(), host(s.vs).copy()


STEPS = [[30, 0, 5, 17], [1, 40, 1, 1], [1, 1, 1, 1], [-3, 1, -100, 1], [2, 1, 33, 0], [1, 1, 1, 1], [1, -41, 1, 15]]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,nkv,hs,block", [(6, 2, 48, 16), (8, 2, 128, 32)])
def test_steps_of_a_server(heads, nkv, hs, block, half):
    """Prompts, single tokens, drafts taken back, a request finished and a new one in its place: every step's tables, cache
    and attention."""
    s = Server(4, heads, nkv, hs, block, 6, half, 60)
    twin, rng = twin_of(s), np.random.default_rng(30)
    for news in STEPS:
        s.fill(rng, news)
        before = floats(s.out, half).reshape(s.n, heads, hs).copy()
        s.step()
        s.check(twin, before, news)


def test_steps_captured_and_replayed():
    """The same step captured into two graphs on a stream of its own (one kernel launch after the other, nothing allocated)
    and replayed in turn: lengths, tables and inputs change on the device."""
    import torch

    s = Server(4, 8, 2, 64, 16, 6, False, 60)
    twin, rng = twin_of(s), np.random.default_rng(31)
    stream = torch.cuda.Stream()
    s.fill(rng, [0, 0, 0, 0])
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            s.step(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        graphs.append(g)
    for i, news in enumerate(STEPS):
        s.fill(rng, news)
        before = floats(s.out, False).reshape(s.n, s.heads, s.hs).copy()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[i % 2].replay()
        torch.cuda.synchronize()
        s.check(twin, before, news)


def test_calls_on_two_streams_at_once():
    """Two servers, a stream and a scratch each, their steps overlapping."""
    import torch

    servers = [Server(4, 8, 2, 64, 16, 6, False, 60) for _ in range(2)]
    twins, rng = [twin_of(s) for s in servers], np.random.default_rng(32)
    streams = [torch.cuda.Stream() for _ in servers]
    for news in STEPS[:4]:
        before = []
        for s in servers:
            s.fill(rng, news)
            before.append(floats(s.out, False).reshape(s.n, s.heads, s.hs).copy())
        torch.cuda.synchronize()
        for s, st in zip(servers, streams):
            s.step(ctypes.c_void_p(st.cuda_stream))
        torch.cuda.synchronize()
        for s, t, b in zip(servers, twins, before):
            s.check(t, b, news)
