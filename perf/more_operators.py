"""What serving a decoder needs around its 4-bit key-value cache, as measurable cases, each through the
package's public entry points on one GPU:

* ``chunk``: attention of chunks of new tokens, of another length for each sequence, over the pages of the
  cache that holds them and what came before (``kv4.Cache4.attend_chunk``);
* ``pages``: page tables and slot maps kept on the GPU: sequences are cut back to given lengths, their pages
  become free, and new tokens get places (``paging.Pages.cut`` and ``grow``);
* ``fork``: the step of a beam search on the caches: rows of the tables go over to other sequences, pages come
  to be shared, and what a sequence will write to becomes its own (``paging.Pages.cut``, ``fork``, ``grow`` and
  ``paging.copy_pages``; ``kv4.Cache4.read`` of each sequence's last page);
* ``select``: the best continuations of a beam search's beams over the vocabulary (``beams.beam_select``).

The rules of the tables. ``table [sequences, width]`` names each sequence's pages in order, -1 past the last,
``lens`` its tokens, ``refs`` how many entries name a page. New tokens take free pages (``refs`` 0) in ascending
order, sequence after sequence. A last page that is partly filled and named elsewhere too is not written to: the
sequence takes a free page for it (before its others) and the page's tokens move there, save for the lowest of
the sequences that share it where all of them grow. If not all new tokens find room nothing changes.

The rules of the selection. A request's candidates are the tokens of each of its beams, with the beam's score
plus the token's log-probability; a beam that has ended has one, the end token at the beam's own score. They are
compared in 64 bits, NaN as -infinity, equals by the lower beam, then the lower token."""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _spread(count, least, most, seed):
    """`count` lengths spread over [least, most], evenly in their logarithm, the longest among them."""
    r = random.Random(seed)
    got = [int(round(math.exp(r.uniform(math.log(least), math.log(most))))) for _ in range(count - 1)]
    got.insert(r.randrange(count), most)
    return got


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def listed():
    return [
        # three short texts read in two goes through a small layer (12 heads of 64): launches and latency
        {"name": "chunk_f32_short", "kind": "chunk", "type": "f32", "q_heads": 12, "kv_heads": 12, "dim": 64,
         "page": 32, "lens": "40,97,33", "new": "5,64,33"},
        # the last piece of a long document, between 16-bit projections: where the matrix rate decides
        {"name": "chunk_bf16_2k", "kind": "chunk", "type": "bf16", "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "lens": "16384", "new": "2048"},
        # pieces of three prompts between int8 projections, whose outputs are f32
        {"name": "chunk_f32_mixed", "kind": "chunk", "type": "f32", "q_heads": 16, "kv_heads": 4, "dim": 128,
         "page": 64, "lens": "4096,1500,777", "new": "512,500,333"},
        # a short question about two long documents: few rows over a long axis
        {"name": "chunk_f16_question", "kind": "chunk", "type": "f16", "q_heads": 24, "kv_heads": 4, "dim": 128,
         "page": 128, "lens": "65536,50001", "new": "32,17"},
        # a scheduler's step: most sequences add one token, some a piece of their prompt, heads of 64
        {"name": "chunk_bf16_batch", "kind": "chunk", "type": "bf16", "q_heads": 15, "kv_heads": 5, "dim": 64,
         "page": 64, "lens": _text(_spread(24, 150, 8192, 3)),
         "new": "1,1,1,128,1,1,1,1,77,1,1,1,1,1,1,111,1,1,1,1,1,1,1,1"},
        # a step of 256 sequences, some give back rejected draft tokens first: latency
        {"name": "pages_step", "kind": "pages", "page": 64, "pages": 16384, "width": 128, "sequences": 256,
         "longest": 8000, "ended": 0, "back": 4, "prompt": 0},
        # a quarter of 512 sequences has ended, prompts take their places
        {"name": "pages_admit", "kind": "pages", "page": 32, "pages": 200000, "width": 512, "sequences": 512,
         "longest": 16000, "ended": 128, "back": 0, "prompt": 4000},
        # one request with four beams: latency
        {"name": "fork_one", "kind": "fork", "page": 64, "kv_heads": 2, "dim": 64, "requests": 1, "beams": 4,
         "longest": 300, "layers": 2},
        # 24 requests with eight beams each, large pages
        {"name": "fork_batch", "kind": "fork", "page": 128, "kv_heads": 8, "dim": 128, "requests": 24, "beams": 8,
         "longest": 3000, "layers": 2},
        # one request with four beams over a small vocabulary: latency
        {"name": "select_one", "kind": "select", "type": "f32", "requests": 1, "beams": 4, "vocab": 32000,
         "ended": False, "first": False, "banned": False},
        # an odd vocabulary, some beams ended, some tokens banned
        {"name": "select_odd", "kind": "select", "type": "f16", "requests": 7, "beams": 5, "vocab": 50001,
         "ended": True, "first": False, "banned": True},
        # 64 requests with eight beams over a large vocabulary
        {"name": "select_batch", "kind": "select", "type": "bf16", "requests": 64, "beams": 8, "vocab": 128000,
         "ended": True, "first": False, "banned": False},
    ]


def draw(rng):
    def upto(least, most):
        return int(round(math.exp(rng.uniform(math.log(least), math.log(max(least, most))))))

    kind = rng.choice(["chunk", "chunk", "chunk", "chunk", "pages", "fork", "select", "select"])
    c = {"kind": kind}
    if kind == "chunk":
        c.update(type=rng.choice(["f32", "bf16", "f16"]), dim=rng.choice([64, 128]), page=rng.choice([32, 64, 96, 128, 256]),
                 kv_heads=rng.choice([1, 2, 3, 4, 5, 8, 12]))
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 7, 8])
        count = upto(1, 24)
        most = {"f32": 2.0e8, "bf16": 8.0e8, "f16": 4.0e8}[c["type"]] / (count * c["q_heads"])  # scores, as the longest
        new = upto(1, min(3000, math.sqrt(most)))
        long = upto(new, max(new, min(60000, most / new)))
        lens = [upto(1, long) for _ in range(count - 1)] + [long]
        c["new"] = _text([min(n, 1 if rng.random() < 0.4 else upto(1, new)) for n in lens[:-1]] + [new])
        c["lens"] = _text(lens)
    elif kind == "pages":
        c.update(page=rng.choice([32, 64, 96, 128, 256]), sequences=upto(1, 700), longest=upto(10, 12000))
        c["width"] = -(-(c["longest"] + 4001) // c["page"]) + rng.randint(0, 20)
        c["ended"] = rng.choice([0, rng.randint(0, c["sequences"])])
        c["back"] = rng.choice([0, 1, 4, 9])
        c["prompt"] = upto(1, 4000)
        c["pages"] = c["sequences"] * c["width"] + rng.randint(0, 3000)
    elif kind == "fork":
        c.update(page=rng.choice([32, 64, 96, 128, 256]), kv_heads=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([64, 128]),
                 requests=upto(1, 24), beams=rng.choice([2, 3, 4, 5, 8]), longest=upto(1, 3000), layers=rng.choice([1, 2, 3]))
        c["layers"] = min(c["layers"], max(1, int(1.3e8 / (c["requests"] * c["beams"] * c["kv_heads"] * c["dim"] * c["page"]))))
    else:
        c.update(type=rng.choice(["f32", "bf16", "f16"]), beams=rng.choice([1, 2, 3, 4, 5, 8, 16]),
                 ended=rng.random() < 0.5, first=rng.random() < 0.2, banned=rng.random() < 0.3)
        c["vocab"] = upto(300, 200000)
        c["requests"] = upto(1, max(1, min(64, int(6.0e7 / (c["beams"] * c["vocab"])))))
    return c


# ------------------------------------------------------------------ what a program has in hand

def _tables(counts, width, spare, g, device):
    """Page tables as an allocator leaves them after a while: pages in no order, -1 past the last."""
    counts = torch.tensor(counts, device=device)
    order = torch.randperm(int(counts.sum()) + spare, generator=g, device=device).to(torch.int32)
    at = torch.arange(width, device=device)
    where = (torch.cumsum(counts, 0) - counts)[:, None] + at
    there = at < counts[:, None]
    return torch.where(there, order[where.clamp_max(len(order) - 1)], torch.full_like(order[:1], -1)).contiguous(), len(order)


def _pool(pages, heads, page, dim, g, device):
    """A cache of random codes with scales around 1: what tokens left there."""
    tb = 512 // dim

    def bytes_of(low, high, *shape):
        return torch.randint(low, high, (pages, heads, *shape), generator=g, device=device).to(torch.uint8)

    return {"k": bytes_of(0, 256, page, dim // 2), "k_scales": bytes_of(123, 128, page // 32, 4, dim // 32, 8),
            "v": bytes_of(0, 256, page // tb, 16, tb, dim // 32), "v_scales": bytes_of(123, 128, page // 32, dim // 32, 32)}


def _refs(table, pages):
    flat = table.flatten().long()
    return torch.bincount(flat[flat >= 0], minlength=pages).to(torch.int32)


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def prepare(case, seed):
    c, kind = case, case["kind"]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    r, sizes = random.Random(seed), random.Random(9)
    s = {"case": c}
    if kind == "chunk":
        lens, new = _numbers(c["lens"]), _numbers(c["new"])
        need = [-(-n // c["page"]) for n in lens]
        s["table"], pages = _tables(need, max(need), 3, g, dev)
        s["pool"] = _pool(pages, c["kv_heads"], c["page"], c["dim"], g, dev)
        # queries, keys and values side by side, as one projection leaves them
        x = torch.randn(sum(new), c["q_heads"] + 2 * c["kv_heads"], c["dim"], generator=g, device=dev)
        s["q"] = x.to(_TYPES[c["type"]])[:, :c["q_heads"]]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["lens"], s["cu"], s["most"], s["most_new"] = _ints(lens, dev), _ints(cu, dev), max(lens), max(new)
    elif kind == "pages":
        n, page = c["sequences"], c["page"]
        lens = [sizes.randint(1, c["longest"]) for _ in range(n)]
        ended = set(sizes.sample(range(n), c["ended"]))
        s["to"] = _ints([0 if i in ended else m - min(m, r.randint(0, c["back"])) for i, m in enumerate(lens)], dev)
        new = [sizes.randint(1, c["prompt"]) if i in ended else 1 for i in range(n)]
        need = [-(-m // page) for m in lens]
        s["table"], pages = _tables(need, c["width"], c["pages"] - sum(need), g, dev)
        s["lens"], s["new"], s["rows"], s["refs"] = _ints(lens, dev), _ints(new, dev), sum(new), _refs(s["table"], pages)
    elif kind == "fork":
        n, w, page = c["requests"] * c["beams"], c["beams"], c["page"]
        per = [sizes.randint(1, c["longest"]) for _ in range(c["requests"])]
        lens = [m for m in per for _ in range(w)]
        width = -(-(c["longest"] + 1) // page)
        # the beams of a request share all but their last pages, as a search leaves them
        table, pages = _tables([-(-m // page) for m in lens], width, n + 5, g, dev)
        last = ((torch.tensor(lens, device=dev) - 1) // page)[:, None]
        first = torch.arange(n, device=dev) // w * w
        s["table"] = torch.where(torch.arange(width, device=dev) < last, table[first], table).contiguous()
        s["refs"], s["lens"] = _refs(s["table"], pages), _ints(lens, dev)
        s["to"], s["one"] = s["lens"].clone(), torch.ones_like(s["lens"])
        # where the next token lies: the page, the tokens before it there
        s["place"], s["held"] = (s["lens"] // page).long()[:, None], s["lens"] % page
        # of each request some beams go on, each other one becomes a copy of one of those
        parents = []
        for q in range(c["requests"]):
            stay = sorted(r.sample(range(w), r.randint(1, max(1, w // 2 + 1))))
            parents += [q * w + (i if i in stay else r.choice(stay)) for i in range(w)]
        s["parents"] = _ints(parents, dev)
        s["pools"] = [_pool(pages, c["kv_heads"], page, c["dim"], g, dev) for _ in range(c["layers"])]
    else:
        b, w, v = c["requests"], c["beams"], c["vocab"]
        x = torch.randn(b * w, v, generator=g, device=dev)
        x = x.mul_(torch.rand(b * w, 1, generator=g, device=dev) * 2 + 1.5)  # some beams are surer than others
        if c["banned"]:
            x[:, torch.randperm(v, generator=g, device=dev)[:v // 10]] = -math.inf
        s["logits"] = x.to(_TYPES[c["type"]])
        s["scores"] = -20.0 - torch.cumsum(torch.rand(b, w, generator=g, device=dev), 1)
        if c["first"]:
            s["scores"][:, 0], s["scores"][:, 1:] = 0.0, -math.inf
        s["done"] = torch.rand(b, w, generator=g, device=dev) < (0.25 if c["ended"] else 0.0)
        s["end"] = v // 3
    return s


# ------------------------------------------------------------------ the plain forms: attention of chunks

def _values(code, byte):
    """f32 of packed codes [..., dim / 2] and scale bytes [..., dim / 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=code.device)
    code = torch.stack((code & 15, code >> 4), -1).flatten(-2)
    scale = (byte.to(torch.int32) << 23).view(torch.float32)
    scale = torch.where(byte == 255, torch.full_like(scale, math.nan), scale)
    return (table[code.int()].reshape(*byte.shape, 32) * scale[..., None]).reshape(code.shape)


def _held(pool, table, page, most):
    """The cache's keys and values [sequences, heads, most, dim] in f32."""
    pages = table.long().clamp_min(0)
    b, w = pages.shape
    k, ks, v, vs = (pool[n][pages] for n in ("k", "k_scales", "v", "v_scales"))
    heads = k.shape[2]
    k = k.permute(0, 2, 1, 3, 4).reshape(b, heads, w * page, -1)[:, :, :most]
    v = v.permute(0, 2, 1, 3, 5, 4, 6).reshape(b, heads, w * page, -1)[:, :, :most]
    ks = ks.permute(0, 2, 1, 3, 6, 4, 5).reshape(b, heads, w * page, -1)[:, :, :most]
    vs = vs.permute(0, 2, 1, 3, 5, 4).reshape(b, heads, w * page, -1)[:, :, :most]
    return _values(k, ks), _values(v, vs)


def _plain_chunk(s):
    c, dev = s["case"], s["q"].device
    lens, cu, most, new = s["lens"].long(), s["cu"].long(), s["most"], s["most_new"]
    k, v = _held(s["pool"], s["table"], c["page"], most)
    b, heads, _, dim = k.shape
    group, n = c["q_heads"] // heads, s["q"].shape[0]
    t, at = torch.arange(new, device=dev), torch.arange(most, device=dev)
    row = (cu[:-1, None] + t).clamp_max(n - 1)  # rows past a chunk's end are left out at the end
    q = s["q"].float()[row].reshape(b, new, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(b, heads, group * new, dim)
    x = (q @ k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(dim)).reshape(b, heads, group, new, most)
    sees = (lens - (cu[1:] - cu[:-1]))[:, None] + t + 1
    x.masked_fill_((at >= sees[..., None])[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    x = x.div_(torch.where(total == 0, torch.ones_like(total), total))
    v = torch.where((at < lens[:, None])[:, None, :, None], v, torch.zeros((), device=dev))
    o = (x.reshape(b, heads, group * new, most) @ v).reshape(b, heads, group, new, dim)
    o = o.permute(0, 3, 1, 2, 4).reshape(b * new, heads * group, dim)
    i = torch.arange(n, device=dev)
    seq = torch.searchsorted(cu, i, right=True) - 1
    return o[seq * new + i - cu[seq]].to(s["q"].dtype)


# ------------------------------------------------------------------ tables

def _plain_cut(s):
    table, lens, refs = s["table"], s["lens"], s["refs"]
    lens.copy_(torch.minimum(lens, s["to"].clamp_min(0)))
    pages = -(-lens // s["case"]["page"])
    leave = (torch.arange(table.shape[1], device=table.device) >= pages[:, None]) & (table >= 0)
    refs.index_add_(0, table.clamp_min(0).flatten(), -leave.flatten().to(torch.int32))
    table.masked_fill_(leave, -1)


def _plain_fork(s):
    s["table"].copy_(s["table"][s["parents"].long()])
    s["lens"].copy_(s["lens"][s["parents"].long()])
    s["refs"].copy_(_refs(s["table"], s["refs"].shape[0]))


def _plain_grow(s, new, rows):
    """cu, slots, at, moves, ok; the tables are brought up to date."""
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["case"]["page"]
    dev, (n, width), i32 = table.device, table.shape, torch.int32
    place, off = lens.long() // page, lens.long() % page
    last = table.gather(1, place.clamp_max(width - 1)[:, None])[:, 0].long()
    shared = (off > 0) & (new > 0) & (last >= 0) & (refs[last.clamp_min(0)] > 1)
    name = torch.where(shared, last, -1 - torch.arange(n, device=dev))  # another for each that shares nothing
    same = name[:, None] == name
    lower = (same & (torch.arange(n, device=dev) < torch.arange(n, device=dev)[:, None])).any(1)
    own_page = shared & (lower | (same.sum(1) != refs[last.clamp_min(0)]))
    before, after = -(-lens.long() // page), -(-(lens.long() + new.long()) // page)
    want = after - before + own_page
    upto = torch.cumsum(want, 0)
    free = (refs == 0).nonzero()[:, 0]
    cu = torch.nn.functional.pad(torch.cumsum(new.long(), 0), (1, 0))
    ok = (upto[-1] <= free.numel()) & (after <= width).all() & (new >= 0).all() & (cu[-1] <= rows)
    free = torch.nn.functional.pad(free, (0, 1), value=0)
    column = torch.arange(width, device=dev)
    takes = torch.where(own_page[:, None] & (column == place[:, None]), 0, column - before[:, None] + own_page[:, None])
    fresh = ((column >= before[:, None]) & (column < after[:, None])) | (own_page[:, None] & (column == place[:, None]))
    fresh &= ok
    page_of = free[((upto - want)[:, None] + takes).clamp(0, free.numel() - 1)]
    old = table.clone()
    table.copy_(torch.where(fresh, page_of.to(i32), table))
    refs.index_add_(0, torch.where(fresh, page_of, 0).flatten(), fresh.flatten().to(i32))
    gone = own_page & ok
    refs.index_add_(0, last.clamp_min(0), -gone.to(i32))
    moved = table.gather(1, place.clamp_max(width - 1)[:, None])[:, 0]
    none = torch.full_like(lens, -1)
    moves = torch.stack((torch.where(gone, last.to(i32), none), torch.where(gone, moved, none),
                         torch.where(gone, off.to(i32), torch.zeros_like(lens))))
    i = torch.arange(rows, device=dev)
    seq = (torch.searchsorted(cu, i, right=True) - 1).clamp(0, n - 1)
    there = (i < cu[-1]) & ok
    at = torch.where(there, lens.long()[seq] + i - cu[seq], -1)
    entry = table[seq, (at // page).clamp(0, width - 1)].long()
    slots = torch.where(there & (entry >= 0), entry * page + at.clamp_min(0) % page, -1)
    lens.add_(torch.where(ok, new, torch.zeros_like(new)))
    return torch.where(ok, cu, 0).to(i32), slots, at.to(i32), moves, ok.to(i32)[None]


def _plain_copy(pool, moves):
    """What holds the tokens that move, 32 at a time."""
    src, dst, tokens = moves.long()
    page = pool["k"].shape[2]
    i, block = ((torch.arange(page // 32, device=src.device) * 32 < tokens[:, None]) & (src >= 0)[:, None]).nonzero().T
    for name in ("k", "k_scales", "v", "v_scales"):
        x = pool[name].view(*pool[name].shape[:2], page // 32, -1)
        x[dst[i], :, block] = x[src[i], :, block]


def _plain_pages(s):
    _plain_cut(s)
    cu, slots, at, moves, ok = _plain_grow(s, s["new"], s["rows"])
    return s["table"], s["lens"], s["refs"], cu, slots, at, moves, ok


def _plain_read(pool, table, held, page):
    k, v = _held(pool, table, page, page)
    there = (torch.arange(page, device=held.device) < held[:, None])[:, None, :, None]
    return torch.where(there, k, torch.zeros_like(k)), torch.where(there, v, torch.zeros_like(v))


def _plain_fork_step(s):
    _plain_cut(s)
    _plain_fork(s)
    cu, slots, at, moves, ok = _plain_grow(s, s["one"], len(s["one"]))
    [_plain_copy(pool, moves) for pool in s["pools"]]
    last = s["table"].gather(1, s["place"])
    return s["table"], s["lens"], s["refs"], slots, moves, ok, \
        [_plain_read(pool, last, s["held"], s["case"]["page"]) for pool in s["pools"]]


# ------------------------------------------------------------------ the selection

def _plain_select(s):
    b, w = s["scores"].shape
    x = s["logits"].float()
    most = min(w, x.shape[1])
    wide = x.double()
    top = wide.amax(-1, keepdim=True)
    total = top + (wide - top).exp_().sum(-1, keepdim=True).log()
    order = x.sort(dim=-1, descending=True, stable=True).indices[:, :most]
    key = s["scores"].double().reshape(-1, 1) + (wide.gather(1, order) - total)
    key = torch.where(key.isnan(), torch.full_like(key, -math.inf), key)
    first = torch.arange(most, device=x.device)
    order = torch.where(key[:, :1] == -math.inf, first, order)  # nothing tells its tokens apart
    done = s["done"].reshape(-1, 1)
    alone = s["scores"].double().reshape(-1, 1)
    alone = torch.where(alone.isnan(), torch.full_like(alone, -math.inf), alone)
    key = torch.where(done, alone, key).reshape(b, -1)
    order = torch.where(done, torch.full_like(order, s["end"]), order).reshape(b, -1)
    out = (done & (first > 0)).reshape(b, -1)  # an ended beam has one candidate
    best = key.sort(dim=-1, descending=True, stable=True).indices
    best = best.gather(1, out.gather(1, best).to(torch.uint8).sort(dim=-1, stable=True).indices)[:, :w]
    parent = torch.div(best, most, rounding_mode="floor")
    token = order.gather(1, best)
    ended = s["done"].gather(1, parent) | (token == s["end"])
    parent = parent + torch.arange(b, device=x.device)[:, None] * w
    return key.gather(1, best).float(), parent.to(torch.int32), token.to(torch.int32), ended


# ------------------------------------------------------------------ one pass

def _handle(s):
    """The tables and caches that a program keeps."""
    if "handle" not in s:
        from borch_amd import kv4, paging
        names = ("k", "k_scales", "v", "v_scales")
        s["caches"] = [kv4.Cache4(*(p[n] for n in names)) for p in s.get("pools", [s.get("pool")]) if p]
        s["handle"] = paging.Pages(s["table"], s["lens"], s["refs"], s["case"]["page"]) if "refs" in s else None
    return s["handle"], s["caches"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "chunk":
        if own:
            _, (cache,) = _handle(s)
            return cache.attend_chunk(s["q"], s["table"], s["lens"], s["cu"], max_len=s["most"])
        return _plain_chunk(s)
    if kind == "pages":
        if own:
            pages, _ = _handle(s)
            pages.cut(s["to"])
            got = pages.grow(s["new"], s["rows"])
            return pages.table, pages.lens, pages.refs, got.cu, got.slots, got.at, got.moves, got.ok
        return _plain_pages(s)
    if kind == "fork":
        if own:
            from borch_amd import paging
            pages, caches = _handle(s)
            pages.cut(s["to"])
            pages.fork(s["parents"])
            got = pages.grow(s["one"], len(s["one"]))
            paging.copy_pages(caches, got.moves)
            last = pages.table.gather(1, s["place"])
            return pages.table, pages.lens, pages.refs, got.slots, got.moves, got.ok, \
                [cache.read(last, s["held"], c["page"]) for cache in caches]
        return _plain_fork_step(s)
    if own:
        from borch_amd import beams
        return tuple(beams.beam_select(s["logits"], s["scores"], s["done"], s["end"]))
    return _plain_select(s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, kind = case, case["kind"]
    size = {"f32": 4}.get(c.get("type"), 2)
    if kind == "chunk":
        lens, new = _numbers(c["lens"]), _numbers(c["new"])
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
        row = c["kv_heads"] * (c["dim"] + c["dim"] // 16)  # a token's keys and values in the cache
        return {"bytes": sum(lens) * row + 2 * sum(new) * c["q_heads"] * c["dim"] * size,
                "flops": 4 * pairs * c["q_heads"] * c["dim"]}
    if kind == "pages":  # lengths; the entries that leave and come; a slot and a place a token
        n, tokens = c["sequences"], c["ended"] * (c["prompt"] + 1) // 2 + c["sequences"] - c["ended"]
        entries = c["ended"] * (c["longest"] // 2 // c["page"] + c["prompt"] // 2 // c["page"] + 2)
        return {"bytes": 28 * n + 12 * entries + 12 * tokens, "flops": 10 * (n + entries + tokens)}
    if kind == "fork":
        n = c["requests"] * c["beams"]
        entries = n * (c["longest"] // 2 // c["page"] + 1)
        tokens = n * c["page"] // 2  # of last pages; about half of them move
        row = c["kv_heads"] * (c["dim"] + c["dim"] // 16)
        return {"bytes": 8 * entries + c["layers"] * (2 * tokens * row + n * c["page"] * 2 * c["kv_heads"] * c["dim"] * 4),
                "flops": 2 * entries + c["layers"] * tokens * row}
    rows = c["requests"] * c["beams"]
    return {"bytes": rows * (c["vocab"] * size + 18), "flops": 3 * rows * c["vocab"]}


# ------------------------------------------------------------------ the definition in 64 bits

_STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_row(pool, which, page, head, off, dim):
    """The f64 values [len(page), dim] of tokens `off` in pages `page` of one head."""
    tb = 512 // dim
    if which == "k":
        code = pool["k"][page, head, off]
        byte = pool["k_scales"][page, head, torch.div(off, 32, rounding_mode="floor"), off.remainder(4)]
        byte = byte.gather(-1, (off.remainder(32) // 4)[:, None, None].expand(-1, dim // 32, 1))[..., 0]
    else:
        code = pool["v"].transpose(3, 4)[page, head, off // tb, off.remainder(tb)].reshape(len(off), -1)
        byte = pool["v_scales"].transpose(3, 4)[page, head, off // 32, off.remainder(32)]
    sign = torch.tensor(_STEPS + tuple(-x for x in _STEPS), dtype=torch.float64, device=code.device)
    x = torch.empty(len(off), dim, dtype=torch.float64, device=code.device)
    x[:, 0::2], x[:, 1::2] = sign[(code % 16).long()], sign[(code // 16).long()]
    return x * torch.pow(2.0, byte.double() - 127.0).repeat_interleave(32, 1)


def exact(case, seed):
    c, kind = case, case["kind"]
    if kind == "pages":  # whole numbers alone
        return None
    s = prepare(case, seed)
    dev = torch.device("cuda")
    if kind == "fork":
        # the values that each sequence's last page holds of its parent's tokens
        page, parents = c["page"], s["parents"].tolist()
        lens, out = s["lens"].tolist(), []
        for pool in s["pools"]:
            k, v = (torch.zeros(len(lens), c["kv_heads"], page, c["dim"], dtype=torch.float64, device=dev) for _ in range(2))
            for i, p in enumerate(parents):
                held = lens[p] % page
                if held:
                    off = torch.arange(held, device=dev)
                    at = s["table"][p, lens[p] // page].long().expand(held)
                    for h in range(c["kv_heads"]):
                        k[i, h, :held] = _exact_row(pool, "k", at, h, off, c["dim"])
                        v[i, h, :held] = _exact_row(pool, "v", at, h, off, c["dim"])
            out.append((k, v))
        return None, None, None, None, None, None, out
    if kind == "select":
        scores = torch.empty(s["scores"].shape, dtype=torch.float64, device=dev)
        for q in range(c["requests"]):
            rows = slice(q * c["beams"], (q + 1) * c["beams"])
            x = torch.log_softmax(s["logits"][rows].double(), -1) + s["scores"][q, :, None].double()
            x[s["done"][q]] = torch.nan
            one = s["scores"][q][s["done"][q]].double()
            every = torch.cat((x[~s["done"][q]].flatten(), one))
            scores[q] = every.topk(c["beams"]).values
        return scores, None, None, None
    lens, new, page, heads, dim = _numbers(c["lens"]), _numbers(c["new"]), c["page"], c["kv_heads"], c["dim"]
    group = c["q_heads"] // heads
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    for b, (n, m) in enumerate(zip(lens, new)):
        rows = slice(int(s["cu"][b]), int(s["cu"][b]) + m)
        at = torch.arange(n, device=dev)
        pages = s["table"][b].long()[at // page]
        hidden = at > (at[n - m:, None])
        for h in range(heads):
            k, v = (_exact_row(s["pool"], which, pages, h, at % page, dim) for which in ("k", "v"))
            kt = k.t().contiguous()
            for j in range(h * group, (h + 1) * group):
                x = torch.mm(s["q"][rows, j].double(), kt) / math.sqrt(dim)
                out[rows, j] = torch.mm(torch.softmax(x.masked_fill_(hidden, -math.inf), -1), v)
    return out
