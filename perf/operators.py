"""Performance cases of the language-model operators: attention over packed prompts, a paged key / value cache held in 8 bits
(append, read back, attention over it) and the cache's pages (fork, truncate, compact).

A case is a dict of plain values; its ``kind`` says which operator it runs:

  prompt   causal attention of whole prompts packed one behind another, grouped heads: ``Backend.attentionPacked``
  append   new tokens quantised into the cache's pages, and the pages that they touched read back: ``KvCache.append``, ``KvCache.read``
  decode   attention of the last one or few tokens of every sequence over its cache: ``KvCache.attention``
  fork     children that share their parent's full pages and own a copy of its part-filled one: ``KvCache.truncate``, ``KvCache.fork``
  compact  live pages moved down into the holes that freed sequences left: ``KvCache.compact``

The cache.  ``k`` / ``v`` [layers][n_pages][kv_heads][page_tokens][head_dim] in 8 bits (``s8``: int8, ``e4m3``: float8_e4m3fn) and one
f32 scale a page and head: a value stands for q * scale.  ``table`` [max_seqs][max_pages] names a sequence's pages, ``lens`` its tokens,
``refs`` the sequences that hold a page (0 = free), ``tail`` the tokens of a sequence's last extension.  The scale of a block (the tokens of
one page, one head) is the smallest power of two, at least 2^-100, with amax <= limit * scale (limit 127 or 448); a block that is added
to keeps its scale or takes a larger one, and what it holds is then rounded again: rn(q * old / new).

``listed()`` are the fixed cases, ``draw(rng)`` gives another one of the same ranges.  With ``own`` false ``run`` computes in plain torch
operations, with ``own`` true it calls the framework.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ESZ = {"f32": 4, "bf16": 2, "f16": 2}
_CACHE = {"s8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def listed():
    return [
        # The smallest prompt: a chat turn of a few tokens, where a launch is most of the time.
        {"name": "prompt_13_tokens", "kind": "prompt", "lens": "13", "heads": 32, "kv_heads": 8, "hd": 128, "x": "bf16"},
        # A batch of prompts as a server packs it: lengths from one token to two thousand, none a multiple of a tile.
        {"name": "prompt_packed_ragged", "kind": "prompt", "lens": "1 77 512 333 1025 2047 17 900 1500", "heads": 32, "kv_heads": 8,
         "hd": 128, "x": "bf16"},
        # One long document.
        {"name": "prompt_8192", "kind": "prompt", "lens": "8192", "heads": 32, "kv_heads": 8, "hd": 128, "x": "bf16"},
        # A small model with seven query heads to a key head, f16, several documents.
        {"name": "prompt_f16_hd64", "kind": "prompt", "lens": "700 1301 259 3001", "heads": 14, "kv_heads": 2, "hd": 64, "x": "f16"},
        # A decode step's append: one token to each of 64 sequences, most of them into a part-filled page.
        {"name": "append_64_tokens", "kind": "append", "old": "4003 1999 17 320 1 77", "new": "1", "seqs": 64, "page": 16, "kv_heads": 8, "hd": 128,
         "cache": "s8", "x": "f32"},
        # Four prompts' keys and values, behind what their sequences hold already (a later turn, a chunk of a long document).
        {"name": "append_prompts", "kind": "append", "old": "0 100 2047 33", "new": "4096 1777 2011 500", "seqs": 4, "page": 64,
         "kv_heads": 8, "hd": 128, "cache": "e4m3", "x": "bf16"},
        # Decoding one short chat: the smallest cache call.
        {"name": "decode_200_tokens", "kind": "decode", "lens": "200", "new": 1, "seqs": 1, "page": 16, "heads": 32, "kv_heads": 8,
         "hd": 128, "cache": "s8", "x": "bf16"},
        # Decoding behind one very long document: few rows, all the work along the sequence.
        {"name": "decode_131000_tokens", "kind": "decode", "lens": "131000", "new": 1, "seqs": 1, "page": 16, "heads": 32, "kv_heads": 8,
         "hd": 128, "cache": "s8", "x": "bf16"},
        # A server's decode step: 48 sequences of very different lengths.
        {"name": "decode_48_ragged", "kind": "decode", "lens": "1 16000 311 9001 64 2500 733 4096", "new": 1, "seqs": 48, "page": 32,
         "heads": 32, "kv_heads": 8, "hd": 128, "cache": "e4m3", "x": "bf16"},
        # Five drafted tokens verified in each of 16 sequences, f32 activations as the GEMVs give them.
        {"name": "decode_5_drafted", "kind": "decode", "lens": "3000 5123 777 2048", "new": 5, "seqs": 16, "page": 64, "heads": 16,
         "kv_heads": 4, "hd": 64, "cache": "s8", "x": "f32"},
        # Beam search or parallel sampling: eight parents, four children each, all layers' part-filled pages copied.
        {"name": "fork_32_beams", "kind": "fork", "lens": "1999 350 777 18 1203 64 5 911", "children": 4, "share": True, "layers": 24,
         "page": 16, "kv_heads": 8, "hd": 128, "cache": "e4m3"},
        # A pool after many sequences have come and gone: the pages in use move into the holes.
        {"name": "compact_3000_pages", "kind": "compact", "pages": 3000, "live": 0.6, "seqs": 40, "layers": 8, "page": 16, "kv_heads": 8,
         "hd": 128, "cache": "e4m3"},
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 5, 7, 8] if kv < 8 else [1, 2, 4]), kv


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "append", "decode", "decode", "fork", "compact"])
    heads, kv = _heads(rng)
    hd, page, cache = rng.choice([64, 128, 128]), rng.choice([16, 32, 64]), rng.choice(["s8", "e4m3"])
    if kind == "prompt":
        n = _log_int(rng, 1, 12)
        return {"kind": kind, "lens": " ".join(str(_log_int(rng, 1, 6000 if n < 3 else 2000)) for _ in range(n)), "heads": heads,
                "kv_heads": kv, "hd": hd, "x": rng.choice(["bf16", "f16"])}
    if kind == "append":
        n = _log_int(rng, 1, 64)
        most = max(1, 8000 // n)
        return {"kind": kind, "old": " ".join(str(rng.choice([0, _log_int(rng, 1, 4000)])) for _ in range(min(n, 6))),
                "new": " ".join(str(_log_int(rng, 1, most)) for _ in range(min(n, 5))), "seqs": n, "page": page, "kv_heads": kv, "hd": hd,
                "cache": cache, "x": rng.choice(["f32", "bf16", "f16"])}
    if kind == "decode":
        n = _log_int(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 3, 4, 6, 8])
        return {"kind": kind, "lens": " ".join(str(_log_int(rng, new, 60000 if n == 1 else 6000)) for _ in range(min(n, 7))), "new": new,
                "seqs": n, "page": page, "heads": heads, "kv_heads": kv, "hd": hd, "cache": cache,
                "x": rng.choice(["f32", "bf16", "f16"])}
    if kind == "fork":
        return {"kind": kind, "lens": " ".join(str(_log_int(rng, 1, 2000)) for _ in range(rng.randint(1, 8))),
                "children": rng.randint(1, 5), "share": rng.random() < 0.7, "layers": rng.randint(1, 16), "page": page, "kv_heads": kv,
                "hd": hd, "cache": cache}
    return {"kind": kind, "pages": _log_int(rng, 200, 3000), "live": rng.choice([0.2, 0.5, 0.8, 0.95]), "seqs": _log_int(rng, 4, 64),
            "layers": rng.randint(1, 8), "page": page, "kv_heads": kv, "hd": hd, "cache": cache}


# -- sizes ---------------------------------------------------------------------------------


def _ints(text):
    return [int(t) for t in str(text).split()]


def _cycled(text, n):
    v = _ints(text)
    return [v[i % len(v)] for i in range(n)]


def _up(a, b):
    return -(-a // b)


# -- inputs --------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _keys(shape, g):
    """Keys or values of real layers: normal, a few channels several times as large as the others."""
    x = torch.randn(shape, device="cuda", generator=g)
    return x.mul_(torch.where(torch.rand(shape[-1], device="cuda", generator=g) < 0.03, 8.0, 1.0))


def _pow2_scale(amax, limit):
    """The smallest power of two, at least 2^-100, with amax <= limit * scale."""
    f, e = torch.frexp(amax.float())
    top, bits = math.frexp(limit)
    e = e - bits + (f > top).to(torch.int32)
    return torch.ldexp(torch.ones_like(f), e.clamp_min(-100))


def _round8(x, cache):
    """Quotients of a value and its scale, rounded to what the cache holds."""
    return torch.round(x).to(torch.int8) if cache == "s8" else x.to(torch.float8_e4m3fn)


def _quantised(shape, g, cache):
    scale, q = [], []
    for _ in range(shape[0]):
        x = _keys(shape[1:], g)
        s = _pow2_scale(x.abs().amax(dim=(-1, -2)), _CACHE[cache][1])
        scale.append(s)
        q.append(_round8(x.div_(s[..., None, None]), cache))
        del x
    return torch.stack(q), torch.stack(scale)


def _make_cache(case, g, lens, layers=1, spare=4, max_seqs=None, room=0):
    """Sequences whose pages lie scattered over the pool, as after some time of serving."""
    page, max_seqs = case["page"], max_seqs or len(lens)
    held = [_up(n, page) for n in lens]
    n_pages, max_pages = sum(held) + spare, max(max(held), 1) + room
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    refs[order[:at].long()] = 1
    shape = (layers, n_pages, case["kv_heads"], page, case["hd"])
    k, ks = _quantised(shape, g, case["cache"])
    v, vs = _quantised(shape, g, case["cache"])
    all_lens = list(lens) + [0] * (max_seqs - len(lens))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table, "lens": _i32(all_lens), "refs": refs,
            "tail": torch.zeros(max_seqs, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "prompt":
        lens, hd, dt = _ints(case["lens"]), case["hd"], _DTYPES[case["x"]]
        total = sum(lens)
        s["q"] = torch.randn((total, case["heads"] * hd), device="cuda", generator=g).mul_(1.5).to(dt)
        s["k"] = _keys((total, case["kv_heads"], hd), g).reshape(total, -1).to(dt)
        s["v"] = _keys((total, case["kv_heads"], hd), g).reshape(total, -1).to(dt)
        s["cu"] = _i32(_offsets(lens))
    elif case["kind"] == "append":
        n, page = case["seqs"], case["page"]
        old, new = _cycled(case["old"], n), _cycled(case["new"], n)
        s["cache"] = _make_cache(case, g, [a + b for a, b in zip(old, new)])
        s["cache"]["tail"].copy_(_i32(new))
        s["seqs"] = _i32(torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist())
        s["cu"] = _i32(_offsets([new[i] for i in s["seqs"].tolist()]))
        first = [old[i] // page * page for i in s["seqs"].tolist()]          # where the first page that is written begins
        back = [old[i] + new[i] - f for i, f in zip(s["seqs"].tolist(), first)]
        s["from"], s["cu_back"], s["back"] = _i32(first), _i32(_offsets(back)), sum(back)
        shape = (sum(new), case["kv_heads"], case["hd"])
        s["k"], s["v"] = (_keys(shape, g).to(_DTYPES[case["x"]]).reshape(shape[0], -1) for _ in range(2))
    elif case["kind"] == "decode":
        n, new = case["seqs"], case["new"]
        lens = _cycled(case["lens"], n)
        s["cache"] = _make_cache(case, g, lens)
        s["seqs"] = _i32(torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist())
        s["cu"], s["longest"] = _i32([new * i for i in range(n + 1)]), max(lens)
        s["q"] = torch.randn((n * new, case["heads"] * case["hd"]), device="cuda", generator=g).mul_(1.5).to(_DTYPES[case["x"]])
    elif case["kind"] == "fork":
        lens, c = _ints(case["lens"]), case["children"]
        parents = len(lens)
        pages = sum(1 if case["share"] else _up(n, case["page"]) for n in lens) * c
        s["cache"] = _make_cache(case, g, lens, case["layers"], spare=pages + 8, max_seqs=parents * (1 + c))
        s["src"] = _i32([p for p in range(parents) for _ in range(c)])
        s["dst"] = _i32([parents + i for i in range(parents * c)])
    else:
        live = int(case["pages"] * case["live"])
        n = min(case["seqs"], live)
        cuts = [live * i // n for i in range(n + 1)]
        lens = [(b - a) * case["page"] - (i * 7) % case["page"] for i, (a, b) in enumerate(zip(cuts, cuts[1:]))]
        s["cache"] = _make_cache(case, g, lens, case["layers"], spare=case["pages"] - live)
        s["table"], s["refs"] = s["cache"]["table"].clone(), s["cache"]["refs"].clone()
    return s


# -- the operators in plain torch ------------------------------------------------------------


def _softmax_rows(scores, visible, v):
    """softmax over the visible places of each row, times v; zero where a row sees nothing."""
    scores.masked_fill_(~visible, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    return p @ v / torch.where(total == 0, 1.0, total)


def _plain_prompt(s):
    case, q, cu = s["case"], s["q"], s["cu"].long()
    hd, kv, group = case["hd"], case["kv_heads"], case["heads"] // case["kv_heads"]
    total, longest, n = q.shape[0], max(_ints(case["lens"])), len(_ints(case["lens"]))
    at = torch.arange(longest, device=q.device)
    rows = (cu[:-1, None] + at).clamp_max(total - 1)                                     # [n][longest]
    qs = q[rows].float().view(n, longest, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, group * longest, hd)
    ks, vs = (t[rows].float().view(n, longest, kv, hd).transpose(1, 2) for t in (s["k"], s["v"]))
    scores = (qs @ ks.transpose(-1, -2)).mul_(hd ** -0.5)
    o = _softmax_rows(scores, (at[None, :] <= at[:, None]).repeat(group, 1), vs)
    o = o.view(n, kv, group, longest, hd).permute(0, 3, 1, 2, 4).reshape(n, longest, -1).to(q.dtype)
    row = torch.arange(total, device=q.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return o[seq, row - cu[seq]]


def _place(cache, seqs, cu, rows):
    """Page and slot of each of the last cu[i + 1] - cu[i] tokens of sequence seqs[i]."""
    row = torch.arange(rows, device=cu.device)
    i = torch.searchsorted(cu, row, right=True) - 1
    pos = cache["lens"].long()[seqs[i]] - (cu[i + 1] - row)
    page = cache["k"].shape[3]
    return cache["table"].long()[seqs[i], pos // page], pos % page


def _plain_append(s):
    case, c, seqs, cu = s["case"], s["cache"], s["seqs"].long(), s["cu"].long()
    rows, kv, hd = s["k"].shape[0], case["kv_heads"], case["hd"]
    pid, slot = _place(c, seqs, cu, rows)
    first = cu[:-1].clamp_max(rows - 1)                       # each sequence's first new token: only its page may hold old ones
    n_pages = c["k"].shape[1]
    for q, scale, x in ((c["k"][0], c["k_scale"][0], s["k"]), (c["v"][0], c["v_scale"][0], s["v"])):
        x = x.float().view(rows, kv, hd)
        amax = torch.full((n_pages, kv), -1.0, device=x.device)
        amax.index_reduce_(0, pid, x.abs().amax(-1), "amax")
        new = _pow2_scale(amax.clamp_min(0), _CACHE[case["cache"]][1])
        p0, f0 = pid[first], slot[first]
        old = scale[p0]
        grown = torch.where(f0[:, None] > 0, torch.maximum(old, new[p0]), new[p0])
        kept = q[p0].float() * (old / grown)[..., None, None]
        keep = torch.arange(q.shape[2], device=x.device)[None, :] < f0[:, None]
        kept = torch.where(keep[:, None, :, None], kept, q[p0].float())
        new[p0] = grown
        scale.copy_(torch.where(amax >= 0, new, scale))
        q[p0] = _round8(kept, case["cache"])
        q[pid, :, slot] = _round8(x / scale[pid][..., None], case["cache"])
    return _plain_read(c, seqs, s["cu_back"].long(), s["from"].long(), s["back"])


def _plain_read(c, seqs, cu, start, rows):
    row = torch.arange(rows, device=cu.device)
    i = torch.searchsorted(cu, row, right=True) - 1
    pos = start[i] + row - cu[i]
    page = c["k"].shape[3]
    pid, slot = c["table"].long()[seqs[i], pos // page], pos % page
    return {n: (c[n][0][pid, :, slot].float() * c[n + "_scale"][0][pid][..., None]).to(torch.bfloat16).reshape(rows, -1)
            for n in ("k", "v")}


def _plain_decode(s):
    case, c, seqs = s["case"], s["cache"], s["seqs"].long()
    n, new, hd, kv = case["seqs"], case["new"], case["hd"], case["kv_heads"]
    group, page = case["heads"] // kv, case["page"]
    lens = c["lens"].long()[seqs]
    pages = c["table"].long()[seqs][:, :_up(s["longest"], page)].clamp_min(0)              # [n][pages]
    ks, vs = ((c[t][0][pages].float() * c[t + "_scale"][0][pages][..., None, None]).transpose(1, 2).reshape(n, kv, -1, hd)
              for t in ("k", "v"))
    q = s["q"].float().view(n, new, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, new * group, hd)
    at = torch.arange(ks.shape[2], device=q.device)
    last = lens[:, None] - new + torch.arange(new, device=q.device)                        # position of each new token
    visible = (at <= last[..., None]).repeat_interleave(group, 1)[:, None]
    o = _softmax_rows((q @ ks.transpose(-1, -2)).mul_(hd ** -0.5), visible, vs.masked_fill_((at >= lens[:, None])[:, None, :, None], 0.0))
    return o.view(n, kv, new, group, hd).transpose(1, 2).reshape(n * new, -1).to(s["q"].dtype)


def _copy_pages(c, src, dst):
    for t in ("k", "v"):
        c[t].view(torch.uint8)[:, dst] = c[t].view(torch.uint8)[:, src]
        c[t + "_scale"][:, dst] = c[t + "_scale"][:, src]


def _free_pages(refs):
    """All pages, the free ones first, each kind by its index."""
    return torch.sort((refs != 0).to(torch.uint8), stable=True).indices


def _held(c, seqs):
    """Which entries of the sequences' rows of the table are pages that they hold."""
    used = (c["lens"].long()[seqs] + c["k"].shape[3] - 1) // c["k"].shape[3]
    return torch.arange(c["table"].shape[1], device=used.device) < used[:, None]


def _plain_fork(s):
    c, src, dst = s["cache"], s["src"].long(), s["dst"].long()
    refs, table, page = c["refs"], c["table"], c["k"].shape[3]
    held = _held(c, dst)                                        # free what the children held
    pages = table[dst].long().clamp_min(0)
    refs.index_add_(0, pages.view(-1), -held.view(-1).to(torch.int32))
    table[dst] = -1
    lens = c["lens"].long()[src]
    held, pages = _held(c, src), table[src].long().clamp_min(0)
    at = torch.arange(table.shape[1], device=src.device)
    copied = held & (at >= lens[:, None] // page) if s["case"]["share"] else held
    number = (copied.view(-1).cumsum(0) - 1).view_as(copied).clamp_min(0)
    fresh = _free_pages(refs)[number]
    taken = torch.where(copied, fresh, pages)
    where = copied.view(-1).nonzero().view(-1)
    _copy_pages(c, pages.view(-1)[where], fresh.view(-1)[where])
    table[dst] = torch.where(held, taken, -1).to(torch.int32)
    refs.index_add_(0, taken.view(-1), held.view(-1).to(torch.int32))
    c["lens"][dst] = lens.to(torch.int32)
    c["tail"][dst] = 0
    return c


def _plain_compact(s):
    c = s["cache"]
    c["table"].copy_(s["table"])                                # the pool with its holes
    c["refs"].copy_(s["refs"])
    refs = c["refs"]
    live = (refs > 0).sum()
    at = torch.arange(refs.numel(), device=refs.device)
    high, low = ((refs > 0) & (at >= live)).nonzero().view(-1), ((refs == 0) & (at < live)).nonzero().view(-1)
    to = at.clone()
    to[high] = low
    _copy_pages(c, high, low)
    refs[low] = refs[high]
    refs[high] = 0
    table = c["table"]
    table.copy_(torch.where(table >= 0, to[table.long().clamp_min(0)].to(torch.int32), table))
    return c


# -- one pass ----------------------------------------------------------------------------------

_be = None


def _backend():
    global _be
    if _be is None:
        from tensorpencil_b200.backend import Backend
        _be = Backend(0)
    return _be


def _kv(s):
    """The framework's handle of the state's cache, made on the first call."""
    if "handle" not in s:
        from tensorpencil_b200.kv_cache import KvCache
        s["handle"] = KvCache.wrap(_backend(), **s["cache"])
    return s["handle"]


def run(s):
    case = s["case"]
    if case["kind"] == "prompt":
        if own:
            return _backend().attentionPacked(s["q"], s["k"], s["v"], s["cu"], case["heads"], case["kv_heads"], case["hd"])
        return _plain_prompt(s)
    if case["kind"] == "append":
        if own:
            kv = _kv(s)
            kv.append(0, s["k"], s["v"], s["seqs"], s["cu"])
            k, v = kv.read(0, s["seqs"], s["cu_back"], s["back"], start=s["from"], dtype=torch.bfloat16)
            return {"k": k, "v": v}
        return _plain_append(s)
    if case["kind"] == "decode":
        if own:
            return _kv(s).attention(0, s["q"], s["seqs"], s["cu"], case["heads"], max_len=s["longest"])
        return _plain_decode(s)
    if case["kind"] == "fork":
        if own:
            kv = _kv(s)
            kv.truncate(s["dst"])
            kv.fork(s["src"], s["dst"], share=case["share"])
            return s["cache"]
        return _plain_fork(s)
    if own:
        s["cache"]["table"].copy_(s["table"])                   # the pool with its holes
        s["cache"]["refs"].copy_(s["refs"])
        _kv(s).compact()
        return s["cache"]
    return _plain_compact(s)


# -- what a pass cannot do without -------------------------------------------------------------


def work(case):
    kv, hd = case["kv_heads"], case["hd"]
    if case["kind"] == "prompt":
        lens = _ints(case["lens"])
        return {"bytes": 2.0 * sum(lens) * hd * 2 * (case["heads"] + kv), "flops": sum(2.0 * n * (n + 1) for n in lens) * hd * case["heads"]}
    if case["kind"] == "append":
        old, new, page = _cycled(case["old"], case["seqs"]), _cycled(case["new"], case["seqs"]), case["page"]
        rows, back = sum(new), sum(a + b - a // page * page for a, b in zip(old, new))
        pages = sum(_up(a + b, page) - a // page for a, b in zip(old, new))
        # the new values read and their bytes written; then the pages read, and written out as bf16
        return {"bytes": 2.0 * kv * (hd * (rows * (_ESZ[case["x"]] + 1) + back * 3) + 8 * pages), "flops": 2.0 * rows * kv * hd}
    if case["kind"] == "decode":
        lens = _cycled(case["lens"], case["seqs"])
        rows = case["seqs"] * case["new"]
        return {"bytes": sum(2.0 * kv * (n * hd + 4 * _up(n, case["page"])) for n in lens) + 2.0 * rows * case["heads"] * hd * _ESZ[case["x"]],
                "flops": sum(4.0 * n for n in lens) * case["new"] * case["heads"] * hd}
    page_bytes = 2.0 * case["layers"] * kv * (case["page"] * hd + 4)
    if case["kind"] == "fork":
        lens, page = _ints(case["lens"]), case["page"]
        copies = sum((n % page > 0) if case["share"] else _up(n, page) for n in lens) * case["children"]
        pages = sum(_up(n, page) for n in lens)
        return {"bytes": 2.0 * copies * page_bytes + 4.0 * pages * (1 + 2 * case["children"]), "flops": 0}
    live = int(case["pages"] * case["live"])
    moved = live * (1 - case["live"])                            # of pages scattered at random, those above the count of live ones
    return {"bytes": 2.0 * moved * page_bytes + 8.0 * live + 8.0 * case["pages"], "flops": 0}


# -- the operators from their definitions, in 64 bits --------------------------------------------


def _attend64(q, k, v, first):
    """q [rows][hd] of consecutive tokens from position `first` on, against k, v [len][hd], all in f64."""
    see = torch.arange(k.shape[0], device=q.device)[None] <= first + torch.arange(q.shape[0], device=q.device)[:, None]
    return torch.softmax(torch.where(see, q @ k.T / math.sqrt(q.shape[1]), -math.inf), dim=-1) @ v


def _exact_prompt(s, case):
    hd, group = case["hd"], case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = s["cu"].tolist()
    for a, b in zip(at, at[1:]):
        for h in range(case["heads"]):
            of = slice(h // group * hd, (h // group + 1) * hd)
            mine = slice(h * hd, (h + 1) * hd)
            out[a:b, mine] = _attend64(s["q"][a:b, mine].double(), s["k"][a:b, of].double(), s["v"][a:b, of].double(), 0)
    return out


def _values64(c, name, seq, n):
    page = c["k"].shape[3]
    pages = c["table"][seq, :_up(n, page)].long()
    x = c[name][0][pages].double() * c[name + "_scale"][0][pages].double()[..., None, None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n]                       # [n][kv_heads][hd]


def _exact_decode(s, case):
    hd, group, new = case["hd"], case["heads"] // case["kv_heads"], case["new"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, seq in enumerate(s["seqs"].tolist()):
        n = int(s["cache"]["lens"][seq])
        k, v = (_values64(s["cache"], t, seq, n) for t in ("k", "v"))
        for h in range(case["heads"]):
            rows = slice(i * new, (i + 1) * new), slice(h * hd, (h + 1) * hd)
            out[rows] = _attend64(s["q"][rows].double(), k[:, h // group], v[:, h // group], n - new)
    return out


def _exact_append(s, case):
    limit, page, c = _CACHE[case["cache"]][1], case["page"], s["cache"]
    at, back = s["cu"].tolist(), {"k": [], "v": []}
    for i, seq in enumerate(s["seqs"].tolist()):
        n, new = int(c["lens"][seq]), at[i + 1] - at[i]
        begin = (n - new) // page * page
        for t in ("k", "v"):
            x = s[t][at[i]:at[i + 1]].double().view(new, case["kv_heads"], case["hd"])
            if n - new > begin:                                    # the page's old values as they stand, ahead of the new ones
                x = torch.cat([_values64(c, t, seq, n - new)[begin:], x])
            pages = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -x.shape[0] % page)).view(-1, page, case["kv_heads"], case["hd"])
            fresh = pages.clone()
            fresh[0, :n - new - begin] = 0                         # a scale covers the new values, and is never less than the old one
            amax = fresh.abs().amax(dim=(1, 3))
            scale = torch.exp2(torch.ceil(torch.log2((amax / limit).clamp_min(2.0 ** -100))))
            if n - new > begin:
                pid = int(c["table"][seq, begin // page])
                scale[0] = torch.maximum(scale[0], c[t + "_scale"][0][pid].double())
            scale = scale[:, None, :, None]
            q = pages / scale
            q = torch.round(q) if case["cache"] == "s8" else q.to(torch.float8_e4m3fn).double()
            back[t].append((q * scale).view(-1, case["kv_heads"] * case["hd"])[:x.shape[0]])
    return {t: torch.cat(back[t]) for t in back}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "prompt":
        return _exact_prompt(s, case)
    if case["kind"] == "decode":
        return _exact_decode(s, case)
    if case["kind"] == "append":
        return _exact_append(s, case)
    return None                                                     # whole numbers, and bytes moved as they are
