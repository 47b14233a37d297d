"""The paged 8-bit cache and the log probabilities as their definitions read, in float64 (numpy, one request after the
other): what the GPU tests compare with."""
import math

import numpy as np


class Tables:
    """The requests' tables, step by step: block ids from a queue's head, blocks given back at its tail."""

    def __init__(self, n_seqs, width, blocks, block, head, free):
        self.tables = np.full((n_seqs, width), -7, np.int64)
        self.lengths = np.zeros(n_seqs, np.int64)
        self.width, self.blocks, self.block, self.head, self.free = width, blocks, block, head, list(free)
        self.ring = np.full(blocks, -9, np.int64)
        for i, b in enumerate(self.free):
            self.ring[(head + i) % blocks] = b

    def step(self, news, n):
        """(status, starts, slots, seq, pos), the state changed where the status is 0."""
        B, S = self.block, len(news)
        up = lambda x: -(-x // B)  # noqa: E731
        nothing = (np.zeros(S + 1, np.int64),) + tuple(np.full(n, -1, np.int64) for _ in range(3))
        after = [max(0, int(l + c)) for l, c in zip(self.lengths, news)]
        if any(a > self.width * B for a in after):
            return (3,) + nothing
        if sum(max(0, int(c)) for c in news) > n:
            return (2,) + nothing
        if sum(max(0, up(a) - up(int(l))) for a, l in zip(after, self.lengths)) > len(self.free):
            return (1,) + nothing
        given, starts, rows = [], [0], []
        for i, (c, a) in enumerate(zip(news, after)):
            before = int(self.lengths[i])
            for b in range(up(before), up(a)):
                self.tables[i, b] = self.free.pop(0)
                self.head = (self.head + 1) % self.blocks
            given += [int(self.tables[i, b]) for b in range(up(a), up(before))]
            for p in range(before, a):
                rows.append((self.tables[i, p // B] * B + p % B, i, p))
            starts.append(starts[-1] + max(0, int(c)))
        for b in given:
            self.ring[(self.head + len(self.free)) % self.blocks] = b
            self.free.append(b)
        self.lengths = np.array(after, np.int64)
        rows += [(-1, -1, -1)] * (n - len(rows))
        return (0, np.array(starts)) + tuple(np.array(x) for x in zip(*rows)) if n else (0, np.array(starts)) + nothing[1:]


def store(cache, scales, x, slots, block):
    """x [n][heads][size] into cache [blocks][heads][block][size] (int8) and scales [blocks][heads] (float32), in place."""
    blocks, heads = scales.shape
    i = 0
    while i < len(slots):
        if not 0 <= slots[i] < blocks * block:
            i += 1
            continue
        page, m = slots[i] // block, 1
        while i + m < len(slots) and 0 <= slots[i + m] < blocks * block and slots[i + m] // block == page:
            m += 1
        held = slots[i] % block
        for h in range(heads):
            run = x[i:i + m, h].astype(np.float64)
            top = np.abs(run).max()  # (numpy's maximum keeps a NaN)
            s = np.float32(top / 127) if np.isfinite(top) else np.float32(np.nan)
            old = scales[page, h] if held else np.float32(0)
            new = s if math.isnan(s) or (not math.isnan(old) and old <= s) else old
            scales[page, h] = new
            if new > old > 0:
                cache[page, h, :held] = np.rint(cache[page, h, :held].astype(np.float64) * np.float64(old) / np.float64(new))
            for t in range(m):
                q = np.rint(run[t] / np.float64(new)) if new > 0 else np.zeros(run.shape[1])
                cache[page, h, slots[i + t] % block] = np.clip(q, -127, 127)  # (of the smallest scales up to 190)
        i += m


def attention(q, kc, ks, vc, vs, tables, starts, lengths, block, group, half=False):
    """(out, bound) of q [n][heads][size] in float64; bound: what an element may be off in float32 arithmetic (see there),
    with float16 queries and outputs where half."""
    n, heads, size = q.shape
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    eps = 2.0 ** -23
    for i in range(len(lengths)):
        length = int(lengths[i])
        rows = int(starts[i + 1] - starts[i])
        page = np.asarray(tables[i][:-(-length // block)], np.int64)
        for h in range(heads):
            kv = h // group
            k = (kc[page, kv].astype(np.float64) * ks[page, kv].astype(np.float64)[:, None, None]).reshape(-1, size)
            v = (vc[page, kv].astype(np.float64) * vs[page, kv].astype(np.float64)[:, None, None]).reshape(-1, size)
            for j in range(rows):
                t, last = starts[i] + j, length - rows + j
                if last < 0:
                    out[t, h] = 0
                    continue
                x = q[t, h].astype(np.float64)
                s = k[:last + 1] @ x / math.sqrt(size)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ v[:last + 1]
                # A score: q in two float16 parts (2^-22 of the row's largest value), then size / 16 instructions for
                # each part, each off by at most 2 eps of the sum of the products' sizes. Its exponent: one rounding of
                # score, value scale and maximum together, and theirs (each below the largest score's and value scale's
                # powers of two together). A weight's
                # relative error is the exponent's (times ln 2) and that of 2^x and of its two float16 parts: 8 eps. The
                # sum: two instructions a unit of 16, at most 2 eps of the sum of sizes each, the same again for the row
                # sum, and a few eps for joining the parts. Every weight's error counts in the sum and in the row sum.
                # A weight's low part is a float16, whose spacing ends at 2^-24: it is off by up to 2^-25 absolutely, on
                # the scale on which the largest p_j times value scale is at least 1 (where the positions that weigh most
                # have values of 0, as integers do, this is what remains).
                a = (np.abs(k[:last + 1]) @ np.full(size, np.abs(x).max()) / math.sqrt(size)).max() * 2 ** -22
                a += (np.abs(k[:last + 1]) @ np.abs(x) / math.sqrt(size)).max() * (size / 8 + 4) * 2 * eps
                top = np.abs(s).max() * 1.45 + np.abs(np.log2(np.clip(vs[page, kv].astype(np.float64), 2.0 ** -100, None))).max()
                weight = a + (2 * top + 48) * eps + 8 * eps
                units = last // 16 + 1
                bound[t, h] = (p @ np.abs(v[:last + 1])) * (2 * weight + (4 * units + 32) * eps)
                integers = np.abs(vc[page, kv].astype(np.float64)).reshape(-1, size)[:last + 1]
                if half:
                    # half a step of float16, 2^-11 of a value at most, once for a weight (the prompts' kernel keeps
                    # float16 requests' weights in one part) and once for the output
                    bound[t, h] += (p @ np.abs(v[:last + 1])) * 2.0 ** -11 + np.abs(out[t, h]) * 2.0 ** -11 + 2.0 ** -25
                bound[t, h] += 2.0 ** -25 * integers.sum(0) * (p * np.repeat(vs[page, kv], block)[:last + 1]).max()
    return out, bound


def logprobs(x, targets, k):
    """(log probability of the targets, entropy, the k largest log probabilities, their ids) in float64."""
    rows, n = x.shape
    chosen, entropy = np.full(rows, np.nan), np.full(rows, np.nan)
    top, ids = np.full((rows, k), np.nan), np.full((rows, k), -1)
    for r in range(rows):
        y = x[r].astype(np.float64)
        if not np.isfinite(y.max()):
            continue
        y = y - y.max()
        with np.errstate(divide="ignore"):
            p = np.exp(y)
            logp = y - math.log(p.sum())
        p = np.exp(logp)
        entropy[r] = -(p[p > 0] * logp[p > 0]).sum()
        if 0 <= targets[r] < n:
            chosen[r] = logp[targets[r]]
        order = np.argsort(-y, kind="stable")[:k]
        top[r], ids[r] = logp[order], order
    return chosen, entropy, top, ids
