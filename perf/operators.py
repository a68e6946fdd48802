"""The paged key / value cache and the attention that reads it: cases, plain forms and
calls, for timing them and for comparing their outputs.

A cache holds the keys and values of many sequences in pages of a pool:

  k, v        [layers, pages, kv_heads, page_size, head_dim]  f16 or bf16
  block_table [sequences, max_blocks] int32, page of each block of a sequence, -1: none
  lengths     [sequences] int32, tokens of each sequence
  refs        [pages] int32, sequences that hold the page, 0: free

Four operators, each with its plain form in elementary torch operations:

  attend   attention of a chunk of new tokens (one token: a decode step) of each
           sequence over all its cached tokens, causal inside the chunk
  append   the new tokens' keys and values written into their sequences' pages
  branch   one step of a search over continuations: the children's old branches are
           freed, parents are forked into them (sharing pages), and each child gets room
           for one more token, a page shared with others being copied first
  compact  the live pages moved, dense and in order, into another pool, with the tables
           rewritten: how a server changes the size of its pool
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "disk-mem-off_b200")

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    glm = dict(heads=96, kv_heads=8, dim=128)  # the GLM-4.7 attention shape of bench.py
    return [
        # a chat with one user: the latency of one token's attention
        dict(name="decode_one", op="attend", dtype="f16", page=64, seqs=1, len_lo=1000,
             len_hi=1000, new_lo=1, new_hi=1, mix=0, **glm),
        # an ordinary decode step of a server: 64 users, contexts of every length
        dict(name="decode_batch", op="attend", dtype="bf16", page=64, seqs=64, len_lo=1,
             len_hi=8192, new_lo=1, new_hi=1, mix=1, **glm),
        # long documents: two contexts of 128 Ki tokens, less one
        dict(name="decode_long", op="attend", dtype="f16", page=128, seqs=2, len_lo=131071,
             len_hi=131071, new_lo=1, new_hi=1, mix=2, **glm),
        # users that decode next to some whose prompts come in chunks
        dict(name="chunk_mixed", op="attend", dtype="bf16", page=32, seqs=33, len_lo=200,
             len_hi=2048, new_lo=1, new_hi=256, mix=3, **glm),
        # the second half of a long prompt
        dict(name="chunk_prefill", op="attend", dtype="f16", page=64, seqs=1, len_lo=8192,
             len_hi=8192, new_lo=4096, new_hi=4096, mix=4, **glm),
        # 64-wide heads without sharing, small pages, odd lengths (the tests' 700 tokens)
        dict(name="chunk_dim64", op="attend", dtype="bf16", page=16, seqs=7, heads=8, kv_heads=8,
             dim=64, len_lo=700, len_hi=1403, new_lo=3, new_hi=700, mix=5),
        # the write of a decode step
        dict(name="append_decode", op="append", dtype="bf16", page=64, seqs=64, kv_heads=8,
             dim=128, len_lo=1, len_hi=4096, new_lo=1, new_hi=1, mix=6),
        # the write of a long prompt's chunks
        dict(name="append_chunk", op="append", dtype="f16", page=64, seqs=5, kv_heads=8, dim=128,
             len_lo=3001, len_hi=9000, new_lo=1500, new_hi=3000, mix=7),
        # four continuations of two prompts
        dict(name="branch_few", op="branch", dtype="f16", page=16, layers=2, kv_heads=2, dim=128,
             parents=2, width=2, len_lo=100, len_hi=500, mix=8),
        # a wide search over sixteen prompts, many layers
        dict(name="branch_wide", op="branch", dtype="bf16", page=64, layers=8, kv_heads=8, dim=128,
             parents=16, width=8, len_lo=500, len_hi=4000, mix=9),
        # a small model's pool after some hours of work
        dict(name="compact_small", op="compact", dtype="f16", page=16, layers=2, kv_heads=2,
             dim=128, seqs=9, len_lo=10, len_hi=700, spare=40, mix=10),
        # a large pool that gives memory back
        dict(name="compact_large", op="compact", dtype="bf16", page=64, layers=8, kv_heads=8,
             dim=128, seqs=24, len_lo=300, len_hi=2500, spare=300, mix=11),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["attend", "attend", "attend", "append", "branch", "compact"])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), page=rng.choice([16, 32, 64, 128]),
             mix=rng.randrange(1 << 30))
    if op == "attend":
        heads, kv_heads, dim = rng.choice([(96, 8, 128), (96, 8, 128), (16, 2, 128), (8, 8, 64),
                                           (12, 4, 64)])
        c.update(heads=heads, kv_heads=kv_heads, dim=dim, seqs=_log(rng, 1, 64))
        if rng.random() < 0.5:  # decode
            hi = _log(rng, 1, min(131072, (1 << 18) // c["seqs"]))
            c.update(new_lo=1, new_hi=1)
        else:  # chunks: the plain form's scores, seqs x new x length, stay in bounds
            c["seqs"] = _log(rng, 1, 24)
            new = _log(rng, 2, 3000)
            hi = _log(rng, new, max(new, min(16384, (1 << 24) // (c["seqs"] * new))))
            if c["seqs"] * new * hi > 1 << 24:
                c["seqs"] = max(1, (1 << 24) // (new * hi))
            c.update(new_lo=rng.randint(1, new), new_hi=new)
        c.update(len_lo=max(c["new_hi"], _log(rng, 1, hi)), len_hi=max(c["new_hi"], hi))
    elif op == "append":
        c.update(kv_heads=rng.choice([2, 8]), dim=rng.choice([64, 128]), seqs=_log(rng, 1, 64))
        new = _log(rng, 1, 16384 // c["seqs"])
        hi = _log(rng, new, new + 4096)
        c.update(new_lo=rng.randint(1, new), new_hi=new, len_lo=new, len_hi=hi)
    elif op == "branch":
        c.update(layers=rng.choice([1, 2, 8]), kv_heads=rng.choice([2, 8]), dim=128,
                 parents=_log(rng, 1, 16), width=_log(rng, 1, 8), len_lo=1,
                 len_hi=_log(rng, 1, 4000))
    else:
        c.update(layers=rng.choice([1, 2, 8]), kv_heads=rng.choice([2, 8]), dim=128,
                 seqs=_log(rng, 1, 24), len_lo=1, len_hi=_log(rng, 1, 2500),
                 spare=rng.randint(0, 300))
    return c


def _sizes(case: dict) -> tuple[list[int], list[int]]:
    """Length and new tokens of each sequence, from the case alone."""
    r = random.Random(case["mix"])
    n = case["parents"] if case["op"] == "branch" else case["seqs"]
    lens = [_log(r, case["len_lo"], case["len_hi"]) for _ in range(n)]
    new = [1] * n
    if "new_hi" in case:
        # most sequences bring little, the first brings the largest chunk
        new = [min(lens[i], _log(r, case["new_lo"], case["new_hi"]) if i else case["new_hi"])
               for i in range(n)]
    return lens, new


def _blocks(tokens: int, page: int) -> int:
    return -(-tokens // page)


# ---------------------------------------------------------------------------- inputs
def _pool(case: dict, layers: int, pages: int, gen: torch.Generator) -> tuple:
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    return tuple(torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(
        _DTYPES[case["dtype"]]) for _ in range(2))


def _i32(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _laid_out(case: dict, lens: list[int], pages: int, rows: int, max_blocks: int,
              seed: int) -> tuple:
    """Table, lengths and refs of sequences 0.. whose pages lie anywhere in the pool."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((rows, max_blocks), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        b = _blocks(n, case["page"])
        table[i, :b] = order[at:at + b].to(torch.int32)
        refs[order[at:at + b]] = 1
        at += b
    lengths = torch.tensor(lens + [0] * (rows - len(lens)), dtype=torch.int32)
    return table.cuda(), lengths.cuda(), refs.cuda()


def prepare(case: dict, seed: int) -> dict:
    lens, new = _sizes(case)
    page = case["page"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    used = sum(_blocks(n, page) for n in lens)
    s: dict = dict(op=case["op"])
    if case["op"] in ("attend", "append"):
        pages = used + used // 8 + 1
        s["k"], s["v"] = _pool(case, 1, pages, gen)
        s["table"], s["lengths"], s["refs"] = _laid_out(
            case, lens, pages, len(lens), max(_blocks(n, page) for n in lens), seed)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["seqs"], s["starts"] = _i32(list(range(len(lens)))), _i32(starts)
        s["longest"], s["most_new"] = max(lens), max(new)  # a scheduler knows both
        if case["op"] == "attend":
            # scores of standard deviation 1.5: attention neither flat nor on one key
            s["q"] = (1.5 * torch.randn((starts[-1], case["heads"], case["dim"]), generator=gen,
                                        device="cuda")).to(dt)
        else:
            s["new_k"], s["new_v"] = (torch.randn(
                (starts[-1], case["kv_heads"], case["dim"]), generator=gen,
                device="cuda").to(dt) for _ in range(2))
    elif case["op"] == "branch":
        kids = case["parents"] * case["width"]
        pages = used + 2 * kids + 8
        s["k"], s["v"] = _pool(case, case["layers"], pages, gen)
        s["table"], s["lengths"], s["refs"] = _laid_out(
            case, lens, pages, case["parents"] + kids, max(_blocks(n + 1, page) for n in lens),
            seed)
        s["parents"] = _i32([i // case["width"] for i in range(kids)])
        s["children"] = _i32([case["parents"] + i for i in range(kids)])
        s["zero"], s["one"] = _i32([0] * kids), _i32([1] * kids)
    else:
        pages = used + case["spare"]
        s["k"], s["v"] = _pool(case, case["layers"], pages, gen)
        s["table"], s["lengths"], s["refs"] = _laid_out(
            case, lens, pages, len(lens), max(_blocks(n, page) for n in lens), seed)
        s["into_k"], s["into_v"] = torch.zeros_like(s["k"][:, :used]), torch.zeros_like(
            s["v"][:, :used])
        s["into_table"] = torch.full_like(s["table"], -1)
        s["into_lengths"] = torch.zeros_like(s["lengths"])
        s["into_refs"] = torch.zeros(used, dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------- plain forms
def _gathered(pool: torch.Tensor, table: torch.Tensor, tokens: int) -> torch.Tensor:
    """[sequences, kv_heads, tokens, dim] in fp32 of one layer's pool."""
    blocks = -(-tokens // pool.shape[2])
    x = pool[table[:, :blocks].clamp(min=0).long()]            # [B, blocks, heads, page, dim]
    x = x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[4])
    return x[:, :, :tokens].float()


def _plain_attend(s: dict) -> torch.Tensor:
    q, starts, seqs = s["q"], s["starts"].long(), s["seqs"].long()
    n, heads, dim = q.shape
    lens = s["lengths"][seqs].long()
    new = starts[1:] - starts[:-1]
    k = _gathered(s["k"][0], s["table"][seqs], s["longest"])
    v = _gathered(s["v"][0], s["table"][seqs], s["longest"])
    group = heads // k.shape[1]
    # the rows of every sequence, padded to the longest chunk
    i = torch.arange(s["most_new"], device=q.device)
    row = (starts[:-1, None] + i).clamp(max=n - 1)             # [B, M]
    qp = q[row].float().reshape(len(seqs), -1, k.shape[1], group, dim)
    qp = qp.permute(0, 2, 3, 1, 4).reshape(len(seqs), k.shape[1], -1, dim)  # [B, kv, group*M, d]
    scores = torch.matmul(qp, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    key = torch.arange(s["longest"], device=q.device)
    last = lens[:, None] - new[:, None] + i                    # last key that row i sees
    hidden = key > last[:, :, None]                            # [B, M, L]
    scores = scores.reshape(len(seqs), k.shape[1], group, s["most_new"], -1)
    scores = scores.masked_fill(hidden[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(dim=-1, keepdim=True)
    p = p.reshape(len(seqs), k.shape[1], -1, s["longest"])
    out = torch.matmul(p, v).reshape(len(seqs), k.shape[1], group, s["most_new"], dim)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(len(seqs), s["most_new"], heads, dim)
    return out[i[None, :] < new[:, None]].to(q.dtype)          # rows of the batch in order


def _plain_append(s: dict) -> tuple:
    starts, seqs, page = s["starts"].long(), s["seqs"].long(), s["k"].shape[3]
    row = torch.arange(s["new_k"].shape[0], device=starts.device)
    e = torch.searchsorted(starts, row, right=True) - 1
    pos = s["lengths"][seqs[e]].long() - (starts[e + 1] - row)
    at = s["table"][seqs[e], pos // page].long()
    s["k"][0][at, :, pos % page] = s["new_k"]
    s["v"][0][at, :, pos % page] = s["new_v"]
    return s["k"], s["v"]


def _plain_truncate(s: dict, seqs: torch.Tensor, lengths: torch.Tensor) -> None:
    page, at = s["k"].shape[3], seqs.long()
    block = torch.arange(s["table"].shape[1], device=at.device)
    rows = s["table"][at]
    keep = (lengths.long() + page - 1) // page
    drop = (rows >= 0) & (block >= keep[:, None])
    gone = rows[drop].long()
    s["refs"].index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    s["table"][at] = torch.where(drop, -1, rows)
    s["lengths"][at] = lengths


def _plain_fork(s: dict, parents: torch.Tensor, children: torch.Tensor) -> None:
    rows = s["table"][parents.long()]
    held = rows[rows >= 0].long()
    s["refs"].index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s["table"][children.long()] = rows
    s["lengths"][children.long()] = s["lengths"][parents.long()]


def _plain_reserve(s: dict, seqs: torch.Tensor, count: torch.Tensor) -> None:
    """Room for count more tokens of each sequence: the lowest free pages, in the order
    of the sequences; a shared page that would be written is replaced by a copy first."""
    page, at = s["k"].shape[3], seqs.long()
    have, more = s["lengths"][at].long(), count.long()
    tail = (have // page).clamp(max=s["table"].shape[1] - 1)
    old = s["table"][at, tail].long()
    shared = (have % page > 0) & (more > 0) & (s["refs"][old.clamp(min=0)] > 1)
    first = (have + page - 1) // page - shared.long()          # first block to fill
    need = (have + more + page - 1) // page - first
    free = torch.nonzero(s["refs"] == 0)[:, 0]
    before = torch.cumsum(need, 0) - need
    block = torch.arange(s["table"].shape[1], device=at.device)
    fill = (block >= first[:, None]) & (block < (first + need)[:, None])
    rank = before[:, None] + block - first[:, None]
    rows = torch.where(fill, free[torch.where(fill, rank, 0)].to(torch.int32), s["table"][at])
    given = rows[fill].long()
    s["refs"].index_add_(0, old[shared], torch.full_like(old[shared], -1, dtype=torch.int32))
    s["refs"][given] = 1
    src, dst = old[shared], rows[shared, tail[shared]].long()
    filled = torch.arange(page, device=at.device) < (have % page)[shared][:, None]
    pair, slot = torch.nonzero(filled, as_tuple=True)          # the rows that hold tokens
    s["k"][:, dst[pair], :, slot] = s["k"][:, src[pair], :, slot]
    s["v"][:, dst[pair], :, slot] = s["v"][:, src[pair], :, slot]
    s["table"][at] = rows
    s["lengths"][at] = (have + more).to(torch.int32)


def _plain_compact(s: dict) -> None:
    live = torch.nonzero(s["refs"] > 0)[:, 0]
    s["into_k"][:, :len(live)] = s["k"][:, live]
    s["into_v"][:, :len(live)] = s["v"][:, live]
    rank = torch.cumsum((s["refs"] > 0).to(torch.int32), 0, dtype=torch.int32) - 1
    table = s["table"]
    s["into_table"].copy_(torch.where(table >= 0, rank[table.clamp(min=0).long()], -1))
    s["into_lengths"].copy_(s["lengths"])
    s["into_refs"].zero_()
    s["into_refs"][:len(live)] = s["refs"][live]


# ---------------------------------------------------------------------------- one pass
def _cache(s: dict, which: str = ""):
    """The program's handle of its cache, made once."""
    if which + "cache" not in s:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from moe_sm100.paged import PagedKVCache
        s[which + "cache"] = PagedKVCache(s[which + "k"], s[which + "v"], s[which + "table"],
                                          s[which + "lengths"], s[which + "refs"])
    return s[which + "cache"]


def run(s: dict):
    if s["op"] == "attend":
        if own:
            return _cache(s).attend(s["q"], s["seqs"], s["starts"])
        return _plain_attend(s)
    if s["op"] == "append":
        if own:
            _cache(s).append(s["new_k"], s["new_v"], s["seqs"], s["starts"])
            return s["k"], s["v"]
        return _plain_append(s)
    if s["op"] == "branch":
        if own:
            cache = _cache(s)
            cache.truncate(s["children"], s["zero"])
            cache.fork(s["parents"], s["children"])
            cache.reserve(s["children"], s["one"])
        else:
            _plain_truncate(s, s["children"], s["zero"])
            _plain_fork(s, s["parents"], s["children"])
            _plain_reserve(s, s["children"], s["one"])
        return s["table"], s["lengths"], s["refs"], s["k"], s["v"]
    if own:
        _cache(s).compact(into=_cache(s, "into_"))
    else:
        _plain_compact(s)
    return s["into_table"], s["into_lengths"], s["into_refs"], s["into_k"], s["into_v"]


# ---------------------------------------------------------------------------- floors
def work(case: dict) -> dict:
    lens, new = _sizes(case)
    page, row = case["page"], case["kv_heads"] * case["dim"] * 2  # bytes of a token's keys
    blocks = [_blocks(n, page) for n in lens]
    if case["op"] == "attend":
        q = sum(new) * case["heads"] * case["dim"] * 2
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
        return dict(bytes=2 * sum(lens) * row + 2 * q + 4 * (sum(blocks) + 3 * len(lens)),
                    flops=4 * pairs * case["heads"] * case["dim"])
    if case["op"] == "append":
        return dict(bytes=4 * sum(new) * row + 4 * sum(blocks), flops=0)
    if case["op"] == "branch":
        w, layers = case["width"], case["layers"]
        kids = case["parents"] * w
        # each child's shared page: its tokens read once per parent, written once per child
        rows = sum((w + 1) * (n % page) for n in lens)
        # the old branch's entries read, the parent's read and the child's written, refs, free map
        tables = 4 * w * sum(3 * b + 1 for b in blocks) + 4 * (sum(blocks) + 2 * kids + 8)
        return dict(bytes=2 * layers * rows * row + tables, flops=0)
    return dict(bytes=4 * case["layers"] * sum(blocks) * page * row + 16 * sum(blocks),
                flops=0)


# ---------------------------------------------------------------------------- in 64 bits
def exact(case: dict, seed: int):
    """The definitions, sequence by sequence and token by token, in 64 bits."""
    s = prepare(case, seed)
    lens, new = _sizes(case)
    page = case["page"]
    table = s["table"].tolist()
    if case["op"] == "attend":
        outs, at = [], 0
        group = case["heads"] // case["kv_heads"]
        for i, (n, m) in enumerate(zip(lens, new)):
            ids = torch.tensor(table[i][:_blocks(n, page)], device="cuda")
            o = torch.empty((m, case["heads"], case["dim"]), dtype=torch.float64, device="cuda")
            below = torch.arange(n - m, n, device="cuda")[:, None] < torch.arange(n, device="cuda")
            for h in range(case["heads"]):
                kk = s["k"][0, ids, h // group].reshape(-1, case["dim"])[:n].double()
                vv = s["v"][0, ids, h // group].reshape(-1, case["dim"])[:n].double()
                x = s["q"][at:at + m, h].double() @ kk.T / math.sqrt(case["dim"])
                x[below] = -math.inf
                o[:, h] = torch.softmax(x, dim=1) @ vv
            outs.append(o)
            at += m
        return torch.cat(outs)
    if case["op"] == "append":
        at = 0
        for i, (n, m) in enumerate(zip(lens, new)):
            for b in range((n - m) // page, _blocks(n, page)):
                lo, hi = max(n - m, b * page), min(n, (b + 1) * page)
                for pool, rows in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
                    x = rows[at + lo - (n - m):at + hi - (n - m)]
                    pool[0, table[i][b], :, lo - b * page:hi - b * page] = x.transpose(0, 1)
            at += m
        return s["k"].double(), s["v"].double()
    if case["op"] == "branch":
        refs, lengths = s["refs"].tolist(), s["lengths"].tolist()
        k, v = s["k"].double(), s["v"].double()
        kids = list(zip(s["parents"].tolist(), s["children"].tolist()))
        for p, c in kids:  # the children start out empty
            table[c], lengths[c] = list(table[p]), lengths[p]
            for x in table[p]:
                if x >= 0:
                    refs[x] += 1
        free = [x for x, r in enumerate(refs) if r == 0]
        held = list(refs)  # a page is shared or not as it was before the call
        for p, c in kids:
            n = lengths[c]
            if n % page and held[table[c][n // page]] > 1:
                x, y = table[c][n // page], free.pop(0)
                for pool in (k, v):
                    pool[:, y, :, :n % page] = pool[:, x, :, :n % page]
                refs[x] -= 1
                refs[y], table[c][n // page] = 1, y
            elif n % page == 0:
                table[c][n // page] = free.pop(0)
                refs[table[c][n // page]] = 1
            lengths[c] = n + 1
        return _i32(table), _i32(lengths), _i32(refs), k, v
    live = [x for x, r in enumerate(s["refs"].tolist()) if r > 0]
    to = {x: y for y, x in enumerate(live)}
    k, v = s["into_k"].double(), s["into_v"].double()
    for x, y in to.items():
        k[:, y], v[:, y] = s["k"][:, x].double(), s["v"][:, x].double()
    refs = [s["refs"].tolist()[x] for x in live] + [0] * (len(s["into_refs"]) - len(live))
    return _i32([[to.get(x, -1) for x in r] for r in table]), s["lengths"], _i32(refs), k, v
