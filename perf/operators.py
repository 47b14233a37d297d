"""The paged 8-bit cache, the attention that reads it and the log probabilities: their measured cases and plain forms.

Kinds of case: "tables" (b200k_block_tables), "cache" (b200k_cache8_store, then b200k_cache8_load of what the touched
blocks hold), "attention" (b200k_cache8_attention), "logprobs" (b200k_logprobs). Sizes are those of this repository's
own shapes (Llama-3-8B: 32 query and 8 key/value heads of 128, 128256 logits; stories15M: 6 heads of 48, 32000 logits;
the prefill configuration: 4 sequences of 2048 tokens, 8 heads of 64; the decode configuration: 64 sequences of 512
to 8192 positions) or generic.
"""
import ctypes
import math
import sys

import torch

own = False
DEVICE = "cuda"


# --------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one greedy step of the bench's 64 sequences: a token each, a few at a block's end, one finished
        {"name": "tables_step_64", "kind": "tables", "seqs": 64, "longest": 8192, "news": 1, "block": 32},
        # a scheduler's step over many requests: prompts of up to some hundred tokens among single tokens
        {"name": "tables_mixed_1000", "kind": "tables", "seqs": 1000, "longest": 4000, "news": 500, "block": 16},
        # the keys and values of one decode step of the 8B shape, one layer
        {"name": "cache_step_64_f32", "kind": "cache", "seqs": 64, "longest": 4096, "news": 1, "block": 32,
         "kv": 8, "size": 128, "half": False},
        # a prompt call's keys and values, one layer: 64 sequences of about 64 new tokens, in float16
        {"name": "cache_prompts_64_f16", "kind": "cache", "seqs": 64, "longest": 4096, "news": 97, "block": 64,
         "kv": 8, "size": 128, "half": True},
        # a few tokens of a small model checked at once (speculation): the smallest call
        {"name": "attention_small_f32", "kind": "attention", "seqs": 3, "shortest": 5, "longest": 333, "news": 4,
         "block": 16, "heads": 6, "kv": 2, "size": 48, "half": False},
        # decode of the 8B shape over ragged contexts (the decode attention configuration)
        {"name": "attention_decode_64_f32", "kind": "attention", "seqs": 64, "shortest": 512, "longest": 8192,
         "news": 1, "block": 32, "heads": 32, "kv": 8, "size": 128, "half": False},
        # one user with a long context: the split over the context carries it
        {"name": "attention_long_1_f16", "kind": "attention", "seqs": 1, "shortest": 131071, "longest": 131071,
         "news": 1, "block": 64, "heads": 32, "kv": 8, "size": 128, "half": True},
        # whole prompts (the prefill configuration), float32
        {"name": "attention_prompts_4_f32", "kind": "attention", "seqs": 4, "shortest": 2048, "longest": 2048,
         "news": 2048, "block": 32, "heads": 8, "kv": 8, "size": 64, "half": False},
        # a prompt block of several sequences over what their caches hold already, float16
        {"name": "attention_blocks_8_f16", "kind": "attention", "seqs": 8, "shortest": 700, "longest": 4500,
         "news": 509, "block": 64, "heads": 32, "kv": 8, "size": 128, "half": True},
        # a small vocabulary, a few rows, the chosen token alone beside its best alternative
        {"name": "logprobs_5_f16", "kind": "logprobs", "rows": 5, "vocab": 32000, "k": 1, "half": True},
        # what an API answers with after a decode step of 64 sequences
        {"name": "logprobs_step_64_f32", "kind": "logprobs", "rows": 64, "vocab": 128256, "k": 20, "half": False},
        # scoring a prompt block: every position's log probability
        {"name": "logprobs_score_512_f32", "kind": "logprobs", "rows": 512, "vocab": 128256, "k": 5, "half": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tables", "cache", "attention", "attention", "logprobs"])
    block = rng.choice([16, 32, 48, 64, 128])
    if kind == "tables":
        return {"kind": kind, "seqs": _log(rng, 1, 1500), "longest": _log(rng, 1, 5000),
                "news": rng.choice([1, _log(rng, 1, 300)]), "block": block}
    if kind == "cache":
        size = rng.choice([16, 48, 64, 80, 128, 256])
        kv = rng.randint(1, 1024 // size) if size < 256 else rng.randint(1, 4)
        seqs, news = _log(rng, 1, 64), _log(rng, 1, 90)
        return {"kind": kind, "seqs": seqs, "longest": _log(rng, 100, 4000), "news": news, "block": block,
                "kv": min(kv, 8), "size": size, "half": rng.random() < 0.5}
    if kind == "logprobs":
        return {"kind": kind, "rows": _log(rng, 1, 400), "vocab": _log(rng, 320, 128256),
                "k": rng.choice([0, 1, 2, 5, 20, 32]), "half": rng.random() < 0.5}
    size, kv = rng.choice([(16, 2), (48, 3), (64, 8), (64, 1), (96, 4), (128, 1), (128, 8), (256, 2)])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    longest = _log(rng, 1, 30000)
    news = rng.choice([1, 1, _log(rng, 1, 600)])
    # no more than the largest listed cases: of positions, and of scores
    most = int(min(64, 2.0e8 / (longest * kv * size), 2.0e8 / (longest * heads * news)))
    if most < 1:
        news, most = 1, max(1, int(2.0e8 / (longest * kv * size)))
    seqs = _log(rng, 1, min(most, 64))
    return {"kind": kind, "seqs": seqs, "shortest": rng.randint(1, longest), "longest": longest, "news": news,
            "block": block, "heads": heads, "kv": kv, "size": size, "half": rng.random() < 0.5}


# -------------------------------------------------------------------------------------------------- the inputs

def _requests(case, order=None):
    """The requests of a step: (lengths with the new tokens, new tokens) on the host. A case has the same requests
    whatever the seed, in another order."""
    g = torch.Generator().manual_seed(1)
    seqs, longest, shortest = case["seqs"], case["longest"], case.get("shortest", 1)
    lengths = torch.randint(shortest, longest + 1, (seqs,), generator=g)
    if case["news"] == 1:
        news = torch.ones(seqs, dtype=torch.long)
    else:
        # half to all of the most that a request adds: prompt blocks, the last one shorter
        news = torch.randint(max(1, case["news"] // 2), case["news"] + 1, (seqs,), generator=g)
        if shortest == longest == case["news"]:
            news = lengths.clone()
    order = torch.arange(seqs) if order is None else torch.randperm(seqs, generator=order)
    return lengths[order], torch.minimum(news, lengths)[order]


def _pages(lengths, block, g):
    """A shuffled pool with a few blocks to spare and the tables of sequences of these lengths: (tables, blocks)."""
    held = (lengths + block - 1) // block
    used, width = int(held.sum()), max(1, int(held.max()))
    blocks = used + 7
    order = torch.randperm(blocks, generator=g)
    column = torch.arange(width)[None, :]
    at = (torch.cumsum(held, 0) - held)[:, None] + column
    tables = torch.where(column < held[:, None], order[at.clamp(max=blocks - 1)], torch.zeros_like(at))
    return tables, blocks


def _tables_state(case, seed):
    g = torch.Generator().manual_seed(1)  # the same requests whatever the seed, in another order
    seqs, block, longest = case["seqs"], case["block"], case["longest"]
    lengths = torch.randint(0, longest + 1, (seqs,), generator=g)
    if case["news"] == 1:
        news = torch.ones(seqs, dtype=torch.long)
    else:
        prompt = torch.rand(seqs, generator=g) < 0.25
        news = torch.where(prompt, torch.randint(1, case["news"] + 1, (seqs,), generator=g), torch.ones(seqs, dtype=torch.long))
    fate = torch.rand(seqs, generator=g)
    news = torch.where(fate < 0.03, -lengths, news)                       # finished: its blocks go back
    news = torch.where((fate >= 0.03) & (fate < 0.06), torch.full_like(news, -2), news)  # two drafts taken back
    news = torch.where((fate >= 0.06) & (fate < 0.1), torch.zeros_like(news), news)      # waiting
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(seqs, generator=g)
    lengths, news = lengths[order], news[order]
    tables, blocks = _pages(lengths.clamp(min=1), block, g)
    width = (longest + case["news"] + block - 1) // block + 1
    wide = torch.zeros(seqs, width, dtype=torch.long)
    wide[:, :tables.shape[1]] = tables
    after = (lengths + news).clamp(min=0)
    take = int(((after + block - 1) // block - (lengths + block - 1) // block).clamp(min=0).sum())
    free = torch.arange(blocks, blocks + take + 11)[torch.randperm(take + 11, generator=g)]
    blocks += take + 11
    head = int(torch.randint(0, blocks, (1,), generator=g))
    ring = torch.zeros(blocks, dtype=torch.long)
    ring[(head + torch.arange(free.numel())) % blocks] = free
    n = int(news.clamp(min=0).sum()) + 5  # a step's buffers have some room
    i32 = lambda x: x.to(torch.int32).to(DEVICE)  # noqa: E731
    empty = lambda *shape: torch.empty(*shape, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return {"tables": i32(wide), "ring": i32(ring), "state": i32(torch.tensor([head, free.numel(), 0, 0])),
            "lengths": i32(lengths), "news": i32(news), "state_out": empty(4), "lengths_out": empty(seqs),
            "starts": empty(seqs + 1), "slots": empty(n), "seq": empty(n), "pos": empty(n),
            "n": n, "seqs": seqs, "width": width, "blocks": blocks, "block": block}


def _cache(blocks, kv, block, size, gd):
    """A pool as the store leaves one: values of about a bell's shape whose largest is 127, a scale for each block and head."""
    values = (torch.randn(blocks, kv, block, size, generator=gd, device=DEVICE) * 34).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.exp(torch.randn(blocks, kv, generator=gd, device=DEVICE) * 0.3) * 0.03
    return values, scales


def _cache_state(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEVICE).manual_seed(seed)
    block, kv, size = case["block"], case["kv"], case["size"]
    lengths, news = _requests(case, g)
    tables, blocks = _pages(lengths, block, g)
    n = int(news.sum())
    starts = torch.cumsum(news, 0) - news
    seq = torch.repeat_interleave(torch.arange(case["seqs"]), news)
    pos = (lengths - news)[seq] + torch.arange(n) - starts[seq]
    page = tables[seq, pos // block]
    # the blocks that these tokens touch, in the order in which they are touched, and all that they hold then
    first = torch.ones(n, dtype=torch.bool)
    first[1:] = page[1:] != page[:-1]
    row = torch.cumsum(first.long(), 0) - 1
    touched = page[first]
    last = torch.ones(n, dtype=torch.bool)
    last[:-1] = first[1:]
    holds = (pos % block)[last] + 1
    held = torch.repeat_interleave(touched * block, holds) + torch.cat([torch.arange(int(h)) for h in holds])
    dt = torch.float16 if case["half"] else torch.float32
    loud = torch.exp(torch.randn(n, kv, 1, generator=gd, device=DEVICE) * 0.5)  # tokens differ in size
    make = lambda: (torch.randn(n, kv, size, generator=gd, device=DEVICE) * loud).to(dt).reshape(n, kv * size)  # noqa: E731
    k, v = make(), make()
    kc, ks = _cache(blocks, kv, block, size, gd)
    vc, vs = _cache(blocks, kv, block, size, gd)
    m = held.numel()
    empty = lambda *shape: torch.empty(*shape, dtype=dt, device=DEVICE)  # noqa: E731
    return {"k": k, "v": v, "kc": kc, "ks": ks, "vc": vc, "vs": vs, "slots": (page * block + pos % block).to(torch.int32).to(DEVICE),
            "held": held.to(torch.int32).to(DEVICE), "k_out": empty(m, kv * size), "v_out": empty(m, kv * size),
            "touched": touched.to(DEVICE), "row": row.to(DEVICE), "n": n, "m": m, "blocks": blocks, "block": block,
            "kv": kv, "size": size, "half": case["half"]}


def _attention_state(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEVICE).manual_seed(seed)
    block, kv, size, heads = case["block"], case["kv"], case["size"], case["heads"]
    lengths, news = _requests(case, g)
    tables, blocks = _pages(lengths, block, g)
    n = int(news.sum())
    starts = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(news, 0)])
    seq = torch.repeat_interleave(torch.arange(case["seqs"]), news)
    pos = (lengths - news)[seq] + torch.arange(n) - starts[seq]
    kc, ks = _cache(blocks, kv, block, size, gd)
    vc, vs = _cache(blocks, kv, block, size, gd)
    dt = torch.float16 if case["half"] else torch.float32
    q = (torch.randn(n, heads * size, generator=gd, device=DEVICE) * 2).to(dt)  # peaked, as trained heads are
    return {"q": q, "kc": kc, "ks": ks, "vc": vc, "vs": vs, "tables": tables.to(torch.int32).to(DEVICE),
            "starts": starts.to(torch.int32).to(DEVICE), "lengths": lengths.to(torch.int32).to(DEVICE),
            "seq": seq.to(DEVICE), "pos": pos.to(DEVICE), "out": torch.empty_like(q), "most": int(news.max()),
            "longest": int(lengths.max()), "n": n, "seqs": case["seqs"], "width": tables.shape[1], "blocks": blocks,
            "block": block, "heads": heads, "kv": kv, "size": size, "half": case["half"]}


def _logprobs_state(case, seed):
    gd = torch.Generator(device=DEVICE).manual_seed(seed)
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    x = torch.randn(rows, vocab, generator=gd, device=DEVICE) * 2.5
    x[:, ::97] += 6 * torch.rand(rows, (vocab + 96) // 97, generator=gd, device=DEVICE)  # a head and a long tail
    if rows > 2:
        x[1, vocab // 3:] = -math.inf                            # a row under a grammar's mask
        x[2, : vocab // 2] = torch.finfo(torch.float16).min      # one masked by a lowest value
    x = x.to(torch.float16 if case["half"] else torch.float32)
    targets = torch.argmax(x.float() - torch.log(-torch.log(torch.rand(rows, vocab, generator=gd, device=DEVICE).clamp_(1e-20, 1 - 1e-7))), 1)
    f32 = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=DEVICE)  # noqa: E731
    return {"x": x, "targets": targets.to(torch.int32), "logprob": f32(rows), "entropy": f32(rows),
            "top": f32(rows, k), "ids": torch.empty(rows, k, dtype=torch.int32, device=DEVICE),
            "rows": rows, "vocab": vocab, "k": k, "half": case["half"]}


def prepare(case, seed):
    make = {"tables": _tables_state, "cache": _cache_state, "attention": _attention_state, "logprobs": _logprobs_state}
    return {"kind": case["kind"], **make[case["kind"]](case, seed)}


# --------------------------------------------------------------------------------------------- the plain forms

def _tables_plain(s):
    block, blocks = s["block"], s["blocks"]
    length, news, head, count = s["lengths"].long(), s["news"].long(), s["state"][0].long(), s["state"][1].long()
    after, fresh = (length + news).clamp(min=0), news.clamp(min=0)
    starts = torch.nn.functional.pad(torch.cumsum(fresh, 0), (1, 0))
    before_b, after_b = (length + block - 1) // block, (after + block - 1) // block
    take, give = (after_b - before_b).clamp(min=0), (before_b - after_b).clamp(min=0)
    take_at, give_at = torch.cumsum(take, 0) - take, torch.cumsum(give, 0) - give
    column = torch.arange(s["width"], device=DEVICE)[None, :]
    taken = (column >= before_b[:, None]) & (column < after_b[:, None])
    source = (head + take_at[:, None] + column - before_b[:, None]) % blocks
    tables = s["tables"].long()
    tables = torch.where(taken, s["ring"].long()[source], tables)
    given = (column >= after_b[:, None]) & (column < before_b[:, None])
    target = (head + count + give_at[:, None] + column - after_b[:, None]) % blocks
    ring = torch.nn.functional.pad(s["ring"], (0, 1))
    ring = ring.scatter(0, torch.where(given, target, blocks).reshape(-1), tables.to(torch.int32).reshape(-1))[:blocks]
    t = torch.arange(s["n"], device=DEVICE)
    live = t < starts[-1]
    seq = torch.searchsorted(starts[1:], t, right=True).clamp(max=s["seqs"] - 1)
    pos = length[seq] + t - starts[seq]
    slots = tables[seq, (pos // block).clamp(0, s["width"] - 1)] * block + pos % block
    state = torch.stack([(head + take.sum()) % blocks, count - take.sum() + give.sum(), torch.zeros_like(head), starts[-1]])
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    gone = torch.full_like(t, -1)
    return (i32(tables), ring, i32(state), i32(after), i32(starts), i32(torch.where(live, slots, gone)),
            i32(torch.where(live, seq, gone)), i32(torch.where(live, pos, gone)))


def _store_plain(cache, scales, x, s):
    block, row, touched = s["block"], s["row"], s["touched"]
    offset = s["slots"].long() % block
    x = x.reshape(s["n"], s["kv"], s["size"]).float()
    count = touched.numel()
    largest = torch.zeros(count, s["kv"], device=DEVICE).index_reduce(0, row, x.abs().amax(-1), "amax")
    begin = torch.full((count,), block, device=DEVICE, dtype=torch.long).index_reduce(0, row, offset, "amin")
    before = torch.where((begin > 0)[:, None], scales[touched], 0)
    after = torch.maximum(before, (largest.double() / 127).float())
    # each value's quotient in 64 bits: it decides on which side of a half the value falls
    step = torch.where(after > 0, after, 1).double()
    held = (torch.arange(block, device=DEVICE) < begin[:, None])[:, None, :, None]
    pages = cache[touched]
    moved = (pages.double() * (before.double())[:, :, None, None] / step[:, :, None, None]).round().to(torch.int8)
    pages = torch.where(held, moved, pages)
    pages[row, :, offset] = (x.double() / step[row][:, :, None]).round().to(torch.int8)
    cache[touched] = pages
    scales[touched] = after


def _load_plain(cache, scales, s):
    held = s["held"].long()
    page, offset = held // s["block"], held % s["block"]
    x = cache[page, :, offset].float() * scales[page][:, :, None]
    return x.reshape(s["m"], -1).to(s["k"].dtype)


def _cache_plain(s):
    _store_plain(s["kc"], s["ks"], s["k"], s)
    _store_plain(s["vc"], s["vs"], s["v"], s)
    return _load_plain(s["kc"], s["ks"], s), _load_plain(s["vc"], s["vs"], s), s["ks"], s["vs"]


def _whole(cache, scales, s):
    """The sequences' rows of the cache, side by side: [sequence][head][position][value]."""
    pages = s["tables"].long()
    x = cache[pages].float() * scales[pages][:, :, :, None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(s["seqs"], s["kv"], -1, s["size"])


def _attention_plain(s):
    seqs, most, kv, size, group = s["seqs"], s["most"], s["kv"], s["size"], s["heads"] // s["kv"]
    seq, pos = s["seq"], s["pos"]
    at = torch.arange(s["n"], device=DEVICE) - s["starts"].long()[seq]
    q = torch.zeros(seqs, most, s["heads"], size, device=DEVICE)
    q[seq, at] = s["q"].float().reshape(s["n"], s["heads"], size)
    q = q.reshape(seqs, most, kv, group, size).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, size)
    scores = torch.matmul(q, _whole(s["kc"], s["ks"], s).transpose(2, 3)) * (1 / math.sqrt(size))
    position = torch.full((seqs, most), -1, device=DEVICE, dtype=torch.long)
    position[seq, at] = pos
    seen = torch.arange(scores.shape[-1], device=DEVICE) <= position[:, :, None]
    scores = scores.reshape(seqs, kv, group, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    scores = scores - scores.amax(-1, keepdim=True).clamp(min=-3e38)
    scores = torch.exp_(scores)
    scores = scores / scores.sum(-1, keepdim=True).clamp(min=1e-38)
    out = torch.matmul(scores.reshape(seqs, kv, group * most, -1), _whole(s["vc"], s["vs"], s))
    out = out.reshape(seqs, kv, group, most, size).permute(0, 3, 1, 2, 4).reshape(seqs, most, -1)
    return out[seq, at].to(s["q"].dtype)


def _logprobs_plain(s):
    x = s["x"].float()
    x = x - x.amax(1, keepdim=True)
    total = torch.exp(x).sum(1, keepdim=True)
    logp = x - torch.log(total)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0).sum(1)
    chosen = logp.gather(1, s["targets"].long()[:, None])[:, 0]
    # the largest, ties to the lowest id: the value's bits in their order above, the id's complement below
    bits = (s["x"].float() + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    keys = (bits << 32) + (0xFFFFFFFF - torch.arange(s["vocab"], device=DEVICE))
    ids = 0xFFFFFFFF - (torch.topk(keys, s["k"], dim=1).values & 0xFFFFFFFF)
    return chosen, entropy, logp.gather(1, ids), ids.to(torch.int32)


# -------------------------------------------------------------------------------------- the framework's own calls

_lib = None


def _abi():
    global _lib
    if _lib is None:
        if "pyodide-llm_b200" not in sys.path:
            sys.path.insert(0, "pyodide-llm_b200")
        from b200fwd import abi

        abi.load()
        _lib = abi
    return _lib


def _own(s):
    abi = _abi()
    lib, stream = abi.load(), torch.cuda.current_stream().cuda_stream
    p = lambda name: s[name].data_ptr()  # noqa: E731
    if s["kind"] == "tables":
        abi.check(lib.b200k_block_tables(
            p("tables"), p("ring"), p("state_out"), p("lengths_out"), p("starts"), p("slots"), p("seq"), p("pos"),
            p("state"), p("lengths"), p("news"), s["seqs"], s["width"], s["blocks"], s["block"], s["n"], stream))
        return (s["tables"], s["ring"], s["state_out"], s["lengths_out"], s["starts"], s["slots"], s["seq"], s["pos"])
    half = 1 if s["half"] else 0
    if s["kind"] == "cache":
        row = s["kv"] * s["size"]
        abi.check(lib.b200k_cache8_store(
            p("kc"), p("ks"), p("vc"), p("vs"), p("k"), p("v"), p("slots"), s["n"], row, row, s["blocks"], s["block"],
            s["kv"], s["size"], half, stream))
        abi.check(lib.b200k_cache8_load(
            p("k_out"), p("v_out"), p("kc"), p("ks"), p("vc"), p("vs"), p("held"), s["m"], row, row, s["blocks"],
            s["block"], s["kv"], s["size"], half, stream))
        return s["k_out"], s["v_out"], s["ks"], s["vs"]
    if s["kind"] == "attention":
        if "scratch" not in s:  # the workspace that a program keeps
            size = ctypes.c_uint64()
            abi.check(lib.b200k_cache8_attention_scratch(s["n"], s["seqs"], s["heads"], s["kv"], s["size"], half,
                                                         ctypes.byref(size)))
            s["scratch"] = torch.empty(max(1, size.value), dtype=torch.uint8, device=DEVICE)
        row = s["heads"] * s["size"]
        abi.check(lib.b200k_cache8_attention(
            p("out"), p("q"), p("kc"), p("ks"), p("vc"), p("vs"), p("tables"), p("starts"), p("lengths"), s["n"],
            s["seqs"], s["width"], s["blocks"], s["block"], s["heads"], s["kv"], s["size"], row, row, half,
            p("scratch"), stream))
        return s["out"]
    abi.check(lib.b200k_logprobs(p("logprob"), p("entropy"), p("top") if s["k"] else None,
                                 p("ids") if s["k"] else None, p("x"), p("targets"), s["rows"], s["vocab"],
                                 s["vocab"], s["k"], half, stream))
    return s["logprob"], s["entropy"], s["top"], s["ids"]


def run(state):
    if own:
        return _own(state)
    plain = {"tables": _tables_plain, "cache": _cache_plain, "attention": _attention_plain, "logprobs": _logprobs_plain}
    return plain[state["kind"]](state)


# ------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * (2 if case["half"] else 4) + case["rows"] * (12 + 8 * case["k"]), "flops": 6 * values}
    if kind == "tables":
        tokens = case["seqs"] * (1 if case["news"] == 1 else 0.7 + 0.25 * case["news"] / 2)
        return {"bytes": int(16 * case["seqs"] + 12 * tokens + 12 * (tokens / case["block"] + 1)), "flops": int(10 * tokens)}
    lengths, news = _requests(case)
    n, value = int(news.sum()), 2 if case["half"] else 4
    if kind == "cache":
        row, block = case["kv"] * case["size"], case["block"]
        held = int((lengths - (lengths - news) // block * block).sum())
        # the new rows read, the blocks' held and new values written, then read and given whole
        return {"bytes": 2 * row * (n * (value + 1) + (held - n) * 1 + held * (1 + value)), "flops": 2 * row * (4 * n + held)}
    pairs = int((news * (lengths - news) + news * (news + 1) // 2).sum())
    row = case["kv"] * case["size"]
    pages = int(((lengths + case["block"] - 1) // case["block"]).sum())
    return {"bytes": int(lengths.sum()) * row * 2 + pages * (8 * case["kv"] + 4) + 2 * n * case["heads"] * case["size"] * value,
            "flops": 4 * case["heads"] * case["size"] * pairs}


# ---------------------------------------------------------------------------- the definitions, in 64 bits

def _exact_cache(s):
    """Block by block as the definition reads: the largest value's 127th part, then every value in units of it."""
    outs, tops = [], []
    for cache, scales, x in ((s["kc"], s["ks"], s["k"]), (s["vc"], s["vs"], s["v"])):
        x = x.double().view(s["n"], s["kv"], s["size"])
        slots, block = s["slots"].long(), s["block"]
        grid = torch.zeros(s["blocks"], block, s["kv"], s["size"], dtype=torch.float64, device=DEVICE)
        grid.view(-1, s["kv"], s["size"])[slots] = x
        is_new = torch.zeros(s["blocks"] * block, dtype=torch.bool, device=DEVICE)
        is_new[slots] = True
        is_new = is_new.view(s["blocks"], block)[s["touched"]]
        grid = grid[s["touched"]]
        old = cache[s["touched"]].double().permute(0, 2, 1, 3) * scales[s["touched"]].double()[:, None, :, None]
        old_scale = torch.where(is_new[:, 0], 0.0, 1.0)[:, None].double() * scales[s["touched"]].double()
        scale = torch.maximum(old_scale, (grid.abs().amax((1, 3)) / 127).float().double())
        value = torch.where(is_new[:, :, None, None], grid, old)
        steps = torch.round(value / scale[:, None, :, None])
        value = (steps * scale[:, None, :, None]).reshape(-1, s["kv"] * s["size"])
        held = s["held"].long()
        where = torch.zeros(s["blocks"], dtype=torch.long, device=DEVICE)
        where[s["touched"]] = torch.arange(s["touched"].numel(), device=DEVICE)
        outs.append(value[where[held // block] * block + held % block])
        whole = scales.double()
        whole[s["touched"]] = scale
        tops.append(whole)
    return outs[0], outs[1], tops[0], tops[1]


def _exact_attention(s):
    out = torch.zeros(s["n"], s["heads"], s["size"], dtype=torch.float64, device=DEVICE)
    group = s["heads"] // s["kv"]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for i in range(s["seqs"]):
        length = lengths[i]
        page = s["tables"][i, : (length + s["block"] - 1) // s["block"]].long()
        for h in range(s["kv"]):
            k = (s["kc"][page, h].double() * s["ks"][page, h].double()[:, None, None]).flatten(0, 1)[:length]
            v = (s["vc"][page, h].double() * s["vs"][page, h].double()[:, None, None]).flatten(0, 1)[:length]
            rows = s["q"][starts[i]:starts[i + 1]].double().view(-1, s["heads"], s["size"])[:, h * group:(h + 1) * group]
            score = torch.einsum("tgd,ld->tgl", rows, k) / math.sqrt(s["size"])
            last = length - rows.shape[0] + torch.arange(rows.shape[0], device=DEVICE)
            score.masked_fill_(torch.arange(length, device=DEVICE)[None, None] > last[:, None, None], -math.inf)
            out[starts[i]:starts[i + 1], h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out.view(s["n"], -1)


def _exact_logprobs(s):
    x = s["x"].double()
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    entropy = torch.special.entr(torch.exp(logp)).sum(1)
    chosen = logp[torch.arange(s["rows"], device=DEVICE), s["targets"].long()]
    order = torch.sort(x, dim=1, descending=True, stable=True)
    ids = order.indices[:, : s["k"]]
    return chosen, entropy, torch.take_along_dim(logp, ids, 1), ids.to(torch.int32)


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers alone
    s = prepare(case, seed)
    return {"cache": _exact_cache, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](s)
