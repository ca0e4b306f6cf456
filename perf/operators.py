"""The attention of a serving transformer as measurable cases, each through the package's public
entry points on one GPU:

* ``prompt``: softmax attention over whole prompts, causal or not, grouped heads, sequences of
  different lengths packed one after another (``attention.prompt_attention``);
* ``append``: keys and values quantized to 4 bits into the pages of a cache, and the values that
  the cache then holds for them (``kv4.Cache4.append`` and ``read``);
* ``attend``: attention of the newest tokens over the 4-bit cache, with or without the running
  sums of what each cached token received (``kv4.Cache4.attend``);
* ``evict``: the tokens that received least leave the cache, the others close up in new pages
  (``kv4.Cache4.evict`` and ``read``).

The cache's form. A value is one of +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} (sign, two bits of exponent, one
of mantissa) times the power of two that 32 neighbouring channels of a token share: 2^(byte - 127),
with the least exponent that takes the largest magnitude to 6 or below (byte >= 1; 255: one of the
32 was not finite and all read as NaN). Rounding is to nearest, ties to the even code. A page holds
``page`` tokens of every key-value head, in four tensors, first the pages, then the heads:

  k         [page, dim / 2]                      channels 2 i, 2 i + 1 in byte i's low and high half
  k_scales  [page / 32, 4, dim / 32, 8]          token 32 a + 4 c + b at [a, b, :, c]
  v         [page / tb, 16, tb, dim / 32]        token tb a + b, channels dim / 16 n ... at [a, n, b], tb = 512 / dim
  v_scales  [page / 32, dim / 32, 32]            token 32 a + b at [a, :, b]

``table [sequences, pages]`` names each sequence's pages in order, ``lens`` its cached tokens."""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _lens(count, least, most, seed):
    """`count` lengths spread over [least, most], evenly in their logarithm, the longest among them."""
    r = random.Random(seed)
    got = [int(round(math.exp(r.uniform(math.log(least), math.log(most))))) for _ in range(count - 1)]
    got.insert(r.randrange(count), most)
    return ",".join(str(n) for n in got)


def listed():
    return [
        # three short texts through a small encoder-sized layer (12 heads of 64): launches and latency
        {"name": "prompt_f32_short", "kind": "prompt", "type": "f32", "causal": True, "q_heads": 12, "kv_heads": 12,
         "dim": 64, "lens": "5,64,33"},
        # two prompts between int8 projections, whose outputs are f32
        {"name": "prompt_f32_2k", "kind": "prompt", "type": "f32", "causal": True, "q_heads": 16, "kv_heads": 4,
         "dim": 128, "lens": "2048,1111"},
        # one long prompt in half the bytes: where the matrix rate decides
        {"name": "prompt_bf16_8k", "kind": "prompt", "type": "bf16", "causal": True, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "lens": "8192"},
        # a batch of unlike lengths, each seeing the whole of its own text, odd head count
        {"name": "prompt_f16_ragged", "kind": "prompt", "type": "f16", "causal": False, "q_heads": 15, "kv_heads": 5,
         "dim": 64, "lens": "1,2999,17,640,129,1,1500,255"},
        # the keys and values of four prompts enter the cache
        {"name": "append_prompt", "kind": "append", "type": "f32", "kv_heads": 8, "dim": 128, "page": 64,
         "lens": "2048,1111,3001,77", "new": "2048,1111,3001,77"},
        # one token of each of 16 sequences enters: the smallest call
        {"name": "append_token", "kind": "append", "type": "bf16", "kv_heads": 8, "dim": 128, "page": 32,
         "lens": _lens(16, 1, 40, 1), "new": ",".join("1" * 16)},
        # single-token decode of one short sequence, 12 heads of 64: latency
        {"name": "attend_one", "kind": "attend", "type": "f32", "q_heads": 12, "kv_heads": 12, "dim": 64, "page": 64,
         "tokens": 1, "lens": "300", "weights": False},
        # batched decode of unlike lengths, four query heads to a key-value head
        {"name": "attend_batch", "kind": "attend", "type": "bf16", "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "tokens": 1, "lens": _lens(64, 200, 16384, 2), "weights": False},
        # two long documents: few rows over a long axis
        {"name": "attend_long", "kind": "attend", "type": "f32", "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 128, "tokens": 1, "lens": "131072,100001", "weights": False},
        # the last 16 tokens of each prompt again, for the sums that an eviction goes by
        {"name": "attend_window", "kind": "attend", "type": "f16", "q_heads": 24, "kv_heads": 4, "dim": 128,
         "page": 64, "tokens": 16, "lens": "4096,2222,9,1025", "weights": True},
        # a batch halves its caches
        {"name": "evict_half", "kind": "evict", "kv_heads": 8, "dim": 128, "page": 64,
         "lens": "4096,4000,3333,2049,2048,1500,4096,2500", "keep": 2048, "recent": 256},
        # two long documents come down to a quarter
        {"name": "evict_long", "kind": "evict", "kv_heads": 8, "dim": 64, "page": 128, "lens": "65536,50001",
         "keep": 16384, "recent": 64},
    ]


def draw(rng):
    def upto(least, most):
        return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))

    kind = rng.choice(["prompt", "prompt", "append", "attend", "attend", "attend", "evict"])
    c = {"kind": kind, "type": rng.choice(["f32", "bf16", "f16"]), "dim": rng.choice([64, 128]),
         "kv_heads": rng.choice([1, 2, 3, 4, 5, 8, 12]), "page": rng.choice([32, 64, 128, 256])}
    if kind == "prompt":
        del c["page"]
        c["causal"] = rng.random() < 0.75
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 7, 8])
        left = 2.0e10 / (c["q_heads"] * c["dim"])  # pairs of tokens
        left = min(left, 4096.0 ** 2 if c["type"] == "f32" else left)
        lens = []
        for _ in range(upto(1, 9)):
            n = min(upto(1, 5000), int(math.sqrt(left)))
            if n:
                lens.append(n)
                left -= n * n
    elif kind == "append":
        count = upto(1, 60)
        most = 12.0e6 / (count * c["kv_heads"] * c["dim"])  # what read returns
        lens = [min(upto(1, 9000), int(most)) for _ in range(count)]
        if rng.random() < 0.5:
            new = ["1"] * len(lens)
        else:
            new = [str(n if rng.random() < 0.5 else rng.randint(1, n)) for n in lens]
        c["new"] = ",".join(new)
    elif kind == "attend":
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 6, 8, 16])
        c["tokens"] = 1 if rng.random() < 0.7 else upto(2, 24)
        c["weights"] = rng.random() < 0.3
        rows = c["tokens"] * (c["q_heads"] // c["kv_heads"])
        count = upto(1, 64)
        most = min(8.0e6, 3.0e8 / rows) / (count * c["kv_heads"])  # scores
        lens = [min(upto(1, 100000), int(most)) for _ in range(count)]
    else:
        del c["type"]
        count = upto(1, 8)
        lens = [upto(40, 30000) for _ in range(count)]
        most = 16.0e6 / (count * c["kv_heads"] * c["dim"])  # what read returns
        c["keep"] = max(1, min(max(lens) // 2, upto(16, 12000), int(most)))
        c["recent"] = rng.randint(0, min(c["keep"], 300))
    c["lens"] = ",".join(str(n) for n in lens)
    return c


# ------------------------------------------------------------------ what a program has in hand

def _numbers(text):
    return [int(n) for n in text.split(",")]


def _tables(lens, page, g, device):
    """Page tables as an allocator leaves them after a while: pages in no order, -1 past the end."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=g, device=device).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def _pool(pages, heads, page, dim, device):
    tb, u8 = 512 // dim, torch.uint8
    return {"k": torch.zeros(pages, heads, page, dim // 2, dtype=u8, device=device),
            "k_scales": torch.ones(pages, heads, page // 32, 4, dim // 32, 8, dtype=u8, device=device),
            "v": torch.zeros(pages, heads, page // tb, 16, tb, dim // 32, dtype=u8, device=device),
            "v_scales": torch.ones(pages, heads, page // 32, dim // 32, 32, dtype=u8, device=device)}


def _rand(shape, g, device, dtype=torch.float32):
    """Activations of a projection: some channels several times larger than the others."""
    x = torch.randn(shape, generator=g, device=device)
    return x.mul_(torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=device))).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind = torch.device("cuda"), case["kind"]
    lens = _numbers(case["lens"])
    heads, dim = case["kv_heads"], case["dim"]
    s = {"case": case, "sizes": lens}
    if kind == "prompt":
        # q, k and v side by side, as one projection leaves them
        n, hq = sum(lens), case["q_heads"]
        x = torch.randn(n, hq + 2 * heads, dim, generator=g, device=dev).to(_TYPES[case["type"]])
        s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:]
        starts = [0]
        for m in lens:
            starts.append(starts[-1] + m)
        s["cu"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        return s
    page = case["page"]
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if kind == "evict":  # the first pages hold what is there, others wait for what stays
        table, pages = _tables(lens + [case["keep"]] * len(lens), page, g, dev)
        s["table"], s["new_table"] = table[:len(lens)].contiguous(), table[len(lens):, :-(-case["keep"] // page)].contiguous()
    else:
        s["table"], pages = _tables(lens, page, g, dev)
    s["pool"] = _pool(pages, heads, page, dim, dev)
    s["most"] = max(lens)
    fill = sum(lens)
    cu = [0]
    for m in lens:
        cu.append(cu[-1] + m)
    if kind != "append":
        put = _slots(s["table"], s["lens"], torch.tensor(cu, device=dev), fill, page)
        _store(s["pool"], _rand((fill, heads, dim), g, dev), _rand((fill, heads, dim), g, dev), put, page)
    if kind == "append":
        new = _numbers(case["new"])
        n = sum(new)
        x = _rand((n, 2 * heads, dim), g, dev, _TYPES[case["type"]])
        s["new_k"], s["new_v"] = x[:, :heads], x[:, heads:]
        starts = [0]
        for m in new:
            starts.append(starts[-1] + m)
        s["cu"], s["new"] = torch.tensor(starts, dtype=torch.int32, device=dev), new
    elif kind == "attend":
        q = torch.randn(len(lens), case["tokens"], case["q_heads"] + 2 * heads, dim, generator=g, device=dev)
        s["q"] = q.to(_TYPES[case["type"]])[:, :, :case["q_heads"]]
        if case["weights"]:
            s["sums"] = torch.rand(len(lens), heads, s["most"], generator=g, device=dev)
    else:
        # sums of softmax weights: many near nothing, some equal
        w = torch.randn(len(lens), heads, s["most"], generator=g, device=dev).mul_(2).exp_()
        s["sums"] = torch.where(w < 0.3, torch.round(w * 64) / 64, w)
    return s


# ------------------------------------------------------------------ the plain forms

def _slots(table, lens, cu, n, page):
    """(page, place in it) of each of the n packed new tokens, the last ones of their sequences."""
    i = torch.arange(n, device=table.device)
    b = torch.searchsorted(cu.long(), i, right=True) - 1
    at = lens.long()[b] - cu.long()[b + 1] + i
    return table.long()[b, at // page], at % page


def _quantized(x):
    """Codes [..., dim] and scale bytes [..., dim / 32] of x."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    peak = g.abs().amax(-1)
    m, e = torch.frexp(peak)
    e = torch.where(m <= 0.75, e - 3, e - 2).clamp_min(-126)
    e = torch.where(peak == 0, torch.full_like(e, -126), e)
    y = torch.ldexp(g.abs(), -e[..., None])
    code = torch.zeros_like(y, dtype=torch.uint8)
    code = code + (y > 0.25) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)
    code = code.to(torch.uint8) + 8 * torch.signbit(g).to(torch.uint8)
    byte = torch.where(torch.isfinite(peak), e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code.reshape(x.shape), byte


def _store(pool, k, v, put, page):
    at, off = put
    n, heads, dim = k.shape
    tb = 512 // dim
    for name, x in (("k", k), ("v", v)):
        code, byte = _quantized(x)
        code = code[..., 0::2] | (code[..., 1::2] << 4)
        if name == "k":
            pool["k"][at, :, off] = code
            pool["k_scales"][at, :, off // 32, off % 4, :, off % 32 // 4] = byte
        else:
            pool["v"][at, :, off // tb, :, off % tb] = code.reshape(n, heads, 16, dim // 32)
            pool["v_scales"][at, :, off // 32, :, off % 32] = byte


def _values(code, byte):
    """f32 of packed codes [..., dim / 2] and scale bytes [..., dim / 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=code.device)
    code = torch.stack((code & 15, code >> 4), -1).flatten(-2)
    scale = (byte.to(torch.int32) << 23).view(torch.float32)
    scale = torch.where(byte == 255, torch.full_like(scale, math.nan), scale)
    x = table[code.int()].reshape(*byte.shape, 32) * scale[..., None]
    return x.reshape(code.shape)


def _held(pool, table, page, most):
    """The cache's keys and values [sequences, heads, most, dim] in f32."""
    pages = table.long().clamp_min(0)
    b, w = pages.shape
    k, ks, v, vs = (pool[n][pages] for n in ("k", "k_scales", "v", "v_scales"))
    heads, dim = k.shape[2], k.shape[-1] * 2
    k = k.permute(0, 2, 1, 3, 4).reshape(b, heads, w * page, -1)[:, :, :most]
    v = v.permute(0, 2, 1, 3, 5, 4, 6).reshape(b, heads, w * page, -1)[:, :, :most]
    ks = ks.permute(0, 2, 1, 3, 6, 4, 5).reshape(b, heads, w * page, -1)[:, :, :most]
    vs = vs.permute(0, 2, 1, 3, 5, 4).reshape(b, heads, w * page, -1)[:, :, :most]
    return _values(k, ks), _values(v, vs)


def _read(pool, table, lens, page, most):
    k, v = _held(pool, table, page, most)
    there = (torch.arange(most, device=table.device) < lens[:, None].long())[:, None, :, None]
    return torch.where(there, k, torch.zeros_like(k)), torch.where(there, v, torch.zeros_like(v))


def _softmax(x, seen):
    """Over the last axis, of what is seen; a row that sees nothing gets zeros."""
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    return x / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(s):
    c = s["case"]
    q, k, v, cu = s["q"].float(), s["k"].float(), s["v"].float(), s["cu"].long()
    b, most, heads, dim = len(s["sizes"]), max(s["sizes"]), c["kv_heads"], c["dim"]
    group, n = c["q_heads"] // heads, q.shape[0]
    t = torch.arange(most, device=q.device)
    at = cu[:-1, None] + t
    there = at < cu[1:, None]
    at = at.clamp_max(n - 1)
    q = q[at].reshape(b, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(b, heads, group * most, dim)
    k = k[at].permute(0, 2, 3, 1).contiguous()
    v = torch.where(there[:, None, :, None], v[at].permute(0, 2, 1, 3), torch.zeros((), device=q.device))
    x = (q @ k).mul_(1.0 / math.sqrt(dim)).reshape(b, heads, group, most, most)
    seen = there[:, None, :].expand(b, most, most)
    if c["causal"]:
        seen = seen & (t <= t[:, None])
    p = _softmax(x, seen[:, None, None])
    o = p.reshape(b, heads, group * most, most) @ v
    o = o.reshape(b, heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(b * most, heads * group, dim)
    row = torch.arange(n, device=q.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return o[seq * most + row - cu[seq]].to(_TYPES[c["type"]])


def _plain_attend(s):
    c = s["case"]
    k, v = _held(s["pool"], s["table"], c["page"], s["most"])
    b, heads, most, dim = k.shape
    tokens, group = c["tokens"], c["q_heads"] // heads
    q = s["q"].float().reshape(b, tokens, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(b, heads, -1, dim)
    x = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(dim)).reshape(b, heads, group, tokens, most)
    at = torch.arange(most, device=k.device)
    end = s["lens"].long()[:, None] - tokens + 1 + torch.arange(tokens, device=k.device)
    p = _softmax(x, (at < end[..., None])[:, None, None])
    v = torch.where((at < s["lens"].long()[:, None])[:, None, :, None], v, torch.zeros((), device=k.device))
    o = p.reshape(b, heads, -1, most) @ v
    o = o.reshape(b, heads, group, tokens, dim).permute(0, 3, 1, 2, 4).reshape(b, tokens, -1, dim).to(s["q"].dtype)
    if not c["weights"]:
        return o
    s["sums"] += p.sum((2, 3))
    return o, s["sums"]


def _plain_evict(s):
    c = s["case"]
    keep, page, pool, sums = c["keep"], c["page"], s["pool"], s["sums"]
    b, heads, most = sums.shape
    tb = 512 // c["dim"]
    at = torch.arange(most, device=sums.device)
    lens = s["lens"].long()[:, None, None]
    order = torch.where(at >= lens - c["recent"], torch.full_like(sums, math.inf), sums)
    order = torch.where(at >= lens, torch.full_like(sums, -math.inf), order)
    wide = torch.nn.functional.pad(order, (0, max(0, keep - most)), value=-math.inf)
    kept = wide.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    left = torch.minimum(lens, torch.full_like(lens, keep))
    kept = torch.where(torch.arange(keep, device=sums.device) < left, kept, torch.full_like(kept, 1 << 30)).sort(-1).values
    there = kept < (1 << 30)
    src = torch.where(there, kept, torch.zeros_like(kept))
    seq = torch.arange(b, device=sums.device)[:, None, None]
    head = torch.arange(heads, device=sums.device)[:, None]
    p, o = s["table"].long()[seq, src // page], src % page
    put = torch.arange(keep, device=sums.device)
    np, no = s["new_table"].long()[:, put // page][:, None], put % page
    pool["k"][np, head, no] = pool["k"][p, head, o]
    pool["k_scales"][np, head, no // 32, no % 4, :, no % 32 // 4] = \
        pool["k_scales"][p, head, o // 32, o % 4, :, o % 32 // 4]
    pool["v"][np, head, no // tb, :, no % tb] = pool["v"][p, head, o // tb, :, o % tb]
    pool["v_scales"][np, head, no // 32, :, no % 32] = pool["v_scales"][p, head, o // 32, :, o % 32]
    weights = torch.where(there, sums.gather(-1, src), torch.zeros((), device=sums.device))
    left = left[:, 0, 0].to(torch.int32)
    return torch.where(there, kept, torch.full_like(kept, -1)).to(torch.int32), weights, left, \
        _read(pool, s["new_table"], left, page, keep)


# ------------------------------------------------------------------ one pass

def _cache(s):
    """The handle that a program keeps."""
    if "cache" not in s:
        from borch_amd import kv4
        p = s["pool"]
        s["cache"] = kv4.Cache4(p["k"], p["k_scales"], p["v"], p["v_scales"])
    return s["cache"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "prompt":
        if own:
            from borch_amd import attention
            return attention.prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"])
        return _plain_prompt(s)
    if kind == "append":
        if own:
            _cache(s).append(s["new_k"], s["new_v"], s["table"], s["lens"], s["cu"])
            return _cache(s).read(s["table"], s["lens"], s["most"])
        put = _slots(s["table"], s["lens"], s["cu"], s["new_k"].shape[0], c["page"])
        _store(s["pool"], s["new_k"], s["new_v"], put, c["page"])
        return _read(s["pool"], s["table"], s["lens"], c["page"], s["most"])
    if kind == "attend":
        if own:
            o = _cache(s).attend(s["q"], s["table"], s["lens"], max_len=s["most"], weights=s.get("sums"))
            return (o, s["sums"]) if c["weights"] else o
        return _plain_attend(s)
    if own:
        kept, weights, left = _cache(s).evict(s["sums"], s["table"], s["lens"], s["new_table"], c["keep"], c["recent"])
        return kept, weights, left, _cache(s).read(s["new_table"], left, c["keep"])
    return _plain_evict(s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind, lens, heads, dim = case["kind"], _numbers(case["lens"]), case["kv_heads"], case["dim"]
    row = heads * (dim + dim // 16)  # a token's keys and values in the cache
    size = {"f32": 4}.get(case.get("type"), 2)
    if kind == "prompt":
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * (2 * case["q_heads"] + 2 * heads) * dim * size,
                "flops": 4 * pairs * case["q_heads"] * dim}
    if kind == "append":
        n = sum(_numbers(case["new"]))  # in, into the cache; then what all hold, out of it, in f32
        return {"bytes": n * (2 * heads * dim * size + row) + sum(lens) * row
                + len(lens) * max(lens) * 2 * heads * dim * 4, "flops": n * 2 * heads * dim}
    if kind == "attend":
        q = len(lens) * case["tokens"] * case["q_heads"] * dim * size
        sums = 8 * heads * sum(lens) if case["weights"] else 0
        return {"bytes": sum(lens) * row + 2 * q + sums, "flops": 4 * sum(lens) * case["tokens"] * case["q_heads"] * dim}
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": sum(lens) * heads * 4 + len(lens) * heads * case["keep"] * (8 + 2 * dim * 4) + kept * 3 * row,
            "flops": sum(lens) * heads}


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


def _exact_held(s, b, head, n, table=None):
    page, at = s["case"]["page"], torch.arange(n, device=s["lens"].device)
    pages = (s["table"] if table is None else table)[b].long()[at // page]
    return tuple(_exact_row(s["pool"], w, pages, head, at % page, s["case"]["dim"]) for w in ("k", "v"))


def _exact_rounded(x):
    """x as the cache holds it, in f64."""
    g = x.double().unflatten(-1, (-1, 32))
    peak = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(peak / 6.0)).clamp_min(-126.0)
    y = g / torch.pow(2.0, e)
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    return (torch.round(y / step) * step * torch.pow(2.0, e)).flatten(-2)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    lens, heads, dim = s["sizes"], case["kv_heads"], case["dim"]
    dev = torch.device("cuda")
    if kind == "prompt":
        group = case["q_heads"] // heads
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
        at = 0
        for n in lens:
            here = slice(at, at + n)
            mask = torch.ones(n, n, dtype=torch.bool, device=dev)
            mask = mask.tril() if case["causal"] else mask
            for h in range(case["q_heads"]):
                q, k, v = s["q"][here, h].double(), s["k"][here, h // group].double(), s["v"][here, h // group].double()
                x = torch.mm(q, k.t().contiguous()) / math.sqrt(dim)
                out[here, h] = torch.mm(torch.softmax(torch.where(mask, x, -math.inf), -1), v)
            at += n
        return out
    if kind == "append":
        most = s["most"]
        k, v = (torch.zeros(len(lens), heads, most, dim, dtype=torch.float64, device=dev) for _ in range(2))
        at = 0
        for b, (n, new) in enumerate(zip(lens, s["new"])):
            for h in range(heads):  # what was there before reads as nothing
                k[b, h, n - new:n] = _exact_rounded(s["new_k"][at:at + new, h])
                v[b, h, n - new:n] = _exact_rounded(s["new_v"][at:at + new, h])
            at += new
        return k, v
    if kind == "attend":
        tokens, group = case["tokens"], case["q_heads"] // heads
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
        sums = s["sums"].double() if case["weights"] else None
        for b, n in enumerate(lens):
            for h in range(heads):
                k, v = _exact_held(s, b, h, n)
                for t in range(tokens):
                    m = n - tokens + 1 + t
                    if m <= 0:
                        continue
                    q = s["q"][b, t, h * group:(h + 1) * group].double()
                    p = torch.softmax(torch.mm(q, k[:m].t().contiguous()) / math.sqrt(dim), -1)
                    out[b, t, h * group:(h + 1) * group] = torch.mm(p, v[:m])
                    if sums is not None:
                        sums[b, h, :m] += p.sum(0)
        return out if sums is None else (out, sums)
    keep, recent = case["keep"], case["recent"]
    weights = torch.zeros(len(lens), heads, keep, dtype=torch.float64, device=dev)
    k, v = (torch.zeros(len(lens), heads, keep, dim, dtype=torch.float64, device=dev) for _ in range(2))
    for b, n in enumerate(lens):
        for h in range(heads):
            w = s["sums"][b, h, :n].double()
            if n <= keep:
                kept = torch.arange(n, device=dev)
            else:
                old = n - recent
                best = torch.argsort(-w[:old], stable=True)[:keep - recent]
                kept = torch.cat((best.sort().values, torch.arange(old, n, device=dev)))
            hk, hv = _exact_held(s, b, h, n)
            k[b, h, :len(kept)], v[b, h, :len(kept)], weights[b, h, :len(kept)] = hk[kept], hv[kept], w[kept]
    return None, weights, None, (k, v)
