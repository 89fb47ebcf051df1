"""Attention over a paged KV cache and the cache's own work, as timed cases.

Every case is one pass of a layer of a serving program that keeps the keys
and values of its sequences in 64-token pages (``HipContext.new_kv_pages``):

* ``prompt``  packed prompts of different lengths: their keys and values are
              written to the pages, then causal grouped-head attention of
              every token (``write_kv_pages_device``,
              ``attention_pages_device``);
* ``batch``   one decode token, or a few drafted ones, of each sequence of a
              batch whose sequences begin with the same cached prefix: the
              new keys and values are written, then attention of the new
              tokens (the same two calls);
* ``write``   keys and values into pages alone (``write_kv_pages_device``);
* ``branch``  one step of a search that keeps the best branches: every branch
              is forked from a chosen parent (often the same one twice), the
              last step's branches are released, and the pages compacted, over
              all layers of a model (``fork``, ``release``, ``compact``).

The pages hold 16-bit keys and values, so the plain form rounds them as the
cache does; queries stay as they come.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
GGML = {"F32": 0, "F16": 1, "BF16": 30}
PAGE = 64  # tokens of a page
MOST_SCORES = 32 * 8192 * 8192  # query heads * queries * keys of the largest case

_context = None


def context():
    """The program's one context on the GPU."""
    global _context
    if _context is None:
        from diskmule_amd import HipContext
        _context = HipContext(0)
    return _context


# --------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------
def listed():
    small = {"query_heads": 32, "kv_heads": 8, "head_dim": 128}
    slide = {"query_heads": 16, "kv_heads": 8, "head_dim": 256}
    full = {"query_heads": 16, "kv_heads": 2, "head_dim": 512}
    return [
        # a short question on its own: latency
        {"name": "prompt_37", "op": "prompt", **small, "lengths": "37", "window": 0, "kv": "BF16", "q": "F32",
         "out": "F32"},
        # prompts of a queue taken together, one of a single token, none a multiple of a page; results feed a
        # projection that takes bf16
        {"name": "prompt_ragged", "op": "prompt", **small, "lengths": "1,640,77,2048,13,333", "window": 0,
         "kv": "BF16", "q": "F32", "out": "BF16"},
        # one long document
        {"name": "prompt_8192", "op": "prompt", **small, "lengths": "8192", "window": 0, "kv": "BF16", "q": "BF16",
         "out": "BF16"},
        # a sliding-window layer over a prompt of several windows
        {"name": "prompt_sliding_4100", "op": "prompt", **slide, "lengths": "4100", "window": 1024, "kv": "F16",
         "q": "F32", "out": "BF16"},
        # one user's decode step, short conversation: the smallest batch
        {"name": "batch_1", "op": "batch", **slide, "sequences": 1, "prefix": 0, "tail": 300, "new": 1, "window": 0,
         "kv": "F16", "q": "F32", "out": "F32"},
        # sixteen users behind one system prompt
        {"name": "batch_16_prefix_8k", "op": "batch", **small, "sequences": 16, "prefix": 8209, "tail": 400, "new": 1,
         "window": 0, "kv": "BF16", "q": "F32", "out": "F32"},
        # sixty-four samples of one long document
        {"name": "batch_64_prefix_32k", "op": "batch", **small, "sequences": 64, "prefix": 32768, "tail": 1000,
         "new": 1, "window": 0, "kv": "BF16", "q": "BF16", "out": "BF16"},
        # drafted tokens of eight users checked at once in a full-attention layer
        {"name": "batch_8_drafted", "op": "batch", **full, "sequences": 8, "prefix": 4001, "tail": 700, "new": 5,
         "window": 0, "kv": "F16", "q": "F32", "out": "F32"},
        # the keys and values of three prompts
        {"name": "write_prompts", "op": "write", "kv_heads": 8, "head_dim": 128, "lengths": "4097,2000,777",
         "new": 0, "kv": "BF16", "src": "F32"},
        # one token of each of 64 sequences
        {"name": "write_decode_64", "op": "write", "kv_heads": 8, "head_dim": 128,
         "lengths": ",".join(str(65 + 13 * i) for i in range(64)), "new": 1, "kv": "BF16", "src": "F32"},
        # four branches of a small model
        {"name": "branch_4", "op": "branch", "kv_heads": 8, "head_dim": 128, "layers": 8, "roots": 4, "length": 200,
         "branches": 4, "kv": "BF16"},
        # sixty-four branches over the layers of a larger one
        {"name": "branch_64", "op": "branch", "kv_heads": 8, "head_dim": 128, "layers": 32, "roots": 16,
         "length": 250, "branches": 64, "kv": "BF16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "batch", "batch", "batch", "write", "branch"])
    kv = rng.choice(["BF16", "BF16", "F16"])
    q = rng.choice(["F32", kv])
    heads = rng.choice([(32, 8, 128), (32, 8, 128), (16, 8, 256), (16, 2, 512), (8, 1, 64), (24, 8, 80)])
    shape = {"query_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2]}
    window = rng.choice([0, 0, 0, 1024])
    if op == "prompt":
        lengths, total = [], _log(rng, 16, 8192)
        while total > 0 and len(lengths) < 16:
            lengths.append(min(total, _log(rng, 1, 8192)))
            total -= lengths[-1]
        return {"op": op, **shape, "lengths": ",".join(map(str, lengths)), "window": window, "kv": kv, "q": q,
                "out": rng.choice(["F32", "BF16", "BF16", kv])}
    if op == "batch":
        sequences, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 8])
        prefix, tail = rng.choice([0, 1, 1, 1]) * _log(rng, 16, 32768), _log(rng, 4, 2048)
        while heads[0] * sequences * new * (prefix + tail + new) > MOST_SCORES // 16:
            sequences, tail = max(1, sequences // 2), max(4, tail // 2)
        return {"op": op, **shape, "sequences": sequences, "prefix": prefix, "tail": tail, "new": new,
                "window": window, "kv": kv, "q": q, "out": rng.choice(["F32", "F32", "BF16", kv])}
    if op == "write":
        n = _log(rng, 1, 64)
        return {"op": op, "kv_heads": heads[1], "head_dim": heads[2],
                "lengths": ",".join(str(_log(rng, 8, 16384 // n)) for _ in range(n)), "new": rng.choice([0, 1, 4]),
                "kv": kv, "src": rng.choice(["F32", kv])}
    roots = _log(rng, 1, 16)
    return {"op": op, "kv_heads": heads[1], "head_dim": heads[2], "layers": _log(rng, 1, 32), "roots": roots,
            "length": PAGE * rng.randint(0, 6) + rng.randint(1, PAGE - 1), "branches": _log(rng, 1, 64), "kv": kv}


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _scale(case):
    # queries of 128 dims and less come unscaled, wider ones from a norm that leaves nothing to scale
    return 1.0 / math.sqrt(case["head_dim"]) if case["head_dim"] <= 128 else 1.0


def _tails(case):
    """Tokens that each sequence of a batch has cached after the prefix: from a quarter of `tail` to all of it."""
    n, tail = case["sequences"], case["tail"]
    return [max(1, tail - (3 * tail // 4) * i // max(1, n - 1)) if n > 1 else tail for i in range(n)]


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _normal(g, kind, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[kind])


def _inputs(case, seed):
    """Every tensor the case reads, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, kvh, hd = case["op"], case["kv_heads"], case["head_dim"]
    if op in ("prompt", "batch"):
        # scores of a standard deviation of about 1.5
        size = 1.5 / (_scale(case) * math.sqrt(hd))
        source = case["q"]  # a layer's projections leave queries, keys and values in one type
    if op == "prompt":
        n = sum(_lengths(case))
        t = {"q": (_normal(g, "F32", n, case["query_heads"], hd) * size).to(TYPES[case["q"]])}
        t["k"], t["v"] = _normal(g, source, n, kvh, hd), _normal(g, source, n, kvh, hd)
        return t
    if op == "batch":
        b, new, tail = case["sequences"], case["new"], max(_tails(case))
        t = {"q": (_normal(g, "F32", b, new, case["query_heads"], hd) * size).to(TYPES[case["q"]])}
        t["k"], t["v"] = _normal(g, source, b, new, kvh, hd), _normal(g, source, b, new, kvh, hd)
        t["prefix_k"], t["prefix_v"] = (_normal(g, case["kv"], case["prefix"], kvh, hd) for _ in range(2))
        t["tail_k"], t["tail_v"] = (_normal(g, case["kv"], b, tail, kvh, hd) for _ in range(2))
        return t
    if op == "write":
        n = sum(min(m, case["new"] or m) for m in _lengths(case))
        return {"k": _normal(g, case["src"], n, kvh, hd), "v": _normal(g, case["src"], n, kvh, hd)}
    pages = case["roots"] * -(-case["length"] // PAGE)
    return {"image": _normal(g, case["kv"], case["layers"], pages, kvh * 2 * hd * PAGE),
            "parents": torch.randint(0, case["roots"], (case["branches"],), generator=g, device="cuda")}


class _Memory:
    """Device memory of the library, for torch.as_tensor."""

    def __init__(self, owner, address, shape):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<i2", "data": (address, False), "version": 2}


def _view(pages, kind, layers, count, elements):
    """The first `count` pages of each layer, as the cache holds them."""
    per = pages.page_capacity()
    whole = torch.as_tensor(_Memory(pages, pages.layer_ptr(0), (layers, per, elements)), device="cuda")
    return whole.view(TYPES[kind])[:, :count]


def _plan(case, pages, tokens):
    return pages.new_plan(case["query_heads"], case["window"] or None, GGML[case["q"]], GGML[case["out"]], tokens)


def prepare(case, seed):
    op, kvh, hd = case["op"], case["kv_heads"], case["head_dim"]
    t = _inputs(case, seed)
    s = {"case": dict(case), "t": t}
    if op == "prompt":
        lengths = _lengths(case)
        t["sequence"] = torch.tensor(np.repeat(np.arange(len(lengths)), lengths), device="cuda")
        t["position"] = torch.tensor(np.concatenate([np.arange(n) for n in lengths]), device="cuda")
        t["o"] = torch.zeros(t["q"].shape, dtype=TYPES[case["out"]], device="cuda")
        counts = lengths
    elif op == "batch":
        t["tails"] = torch.tensor(_tails(case), device="cuda")
        t["o"] = torch.zeros(t["q"].shape, dtype=TYPES[case["out"]], device="cuda")
    elif op == "write":
        lengths = _lengths(case)
        counts = [min(n, case["new"] or n) for n in lengths]
        first = np.concatenate([[0], np.cumsum([-(-n // PAGE) for n in lengths])])
        at = [np.arange(n - c, n) for n, c in zip(lengths, counts)]
        t["page"] = torch.tensor(np.concatenate([f + p // PAGE for f, p in zip(first, at)]), device="cuda")
        t["slot"] = torch.tensor(np.concatenate([p % PAGE for p in at]), device="cuda")
        s["pages_used"] = int(first[-1])
        if not own:
            t["pool"] = torch.zeros(s["pages_used"], kvh, 2, hd * PAGE, dtype=TYPES[case["kv"]], device="cuda")
    else:
        per = -(-case["length"] // PAGE)
        s["parents"] = [int(p) for p in t["parents"].tolist()]
        s["pages_used"] = case["roots"] * per + case["branches"]
        t["last"] = (t["parents"] + 1) * per - 1
        if not own:
            t["pool"] = torch.zeros(case["layers"], s["pages_used"] + case["branches"], kvh * 2 * hd * PAGE,
                                    dtype=TYPES[case["kv"]], device="cuda")
            t["pool"][:, :case["roots"] * per] = t["image"]
    torch.cuda.synchronize()
    if not own:
        return s
    ctx = s["ctx"] = context()
    if op == "batch":
        _fill_batch(case, s)
    elif op == "branch":
        pages = s["pages"] = ctx.new_kv_pages(GGML[case["kv"]], case["layers"], kvh, hd, case["length"],
                                              s["pages_used"] + case["branches"],
                                              case["roots"] + 2 * case["branches"])
        s["roots"] = [pages.new_sequence() for _ in range(case["roots"])]
        pages.extend(s["roots"], [case["length"]] * case["roots"])
        for layer in range(case["layers"]):  # a cache brought back from where it was saved
            ctx.copy_device(pages.layer_ptr(layer), t["image"][layer].data_ptr(),
                            t["image"][layer].numel() * t["image"].element_size())
        s["live"] = pages.fork([s["roots"][p] for p in s["parents"]], [case["length"]] * case["branches"])
        s["view"] = _view(pages, case["kv"], case["layers"], s["pages_used"], kvh * 2 * hd * PAGE)
    else:
        used = sum(-(-n // PAGE) for n in lengths)
        pages = s["pages"] = ctx.new_kv_pages(GGML[case["kv"]], 1, kvh, hd, max(lengths), used, len(lengths))
        seqs = [pages.new_sequence() for _ in lengths]
        pages.extend(seqs, lengths)
        if op == "prompt":
            s["plan"] = _plan(case, pages, sum(counts))
        else:
            s["plan"] = pages.new_plan(kvh, None, 0, 0, sum(counts))
            s["view"] = _view(pages, case["kv"], 1, used, kvh * 2 * hd * PAGE)[0].view(used, kvh, 2, hd * PAGE)
        s["plan"].set(seqs, counts)
    ctx.synchronize()
    return s


def _fill_batch(case, s):
    """The batch's cache before the step: one prefix, forked, and each sequence's own tokens."""
    ctx, t, kvh, hd, b = s["ctx"], s["t"], case["kv_heads"], case["head_dim"], case["sequences"]
    tails, new, prefix = _tails(case), case["new"], case["prefix"]
    kind, width = GGML[case["kv"]], kvh * hd
    longest = prefix + max(tails) + new
    pages = s["pages"] = ctx.new_kv_pages(kind, 1, kvh, hd, longest,
                                          -(-prefix // PAGE) + b * (-(-(max(tails) + new) // PAGE) + 1), b + 1)
    fill = _plan(case, pages, max(prefix, sum(tails)))
    root = pages.new_sequence()
    if prefix:
        pages.extend([root], [prefix])
        fill.set([root], [prefix])
        ctx.write_kv_pages_device(fill, 0, kind, t["prefix_k"].data_ptr(), width, t["prefix_v"].data_ptr(), width)
    seqs = pages.fork([root] * b, [prefix] * b)
    pages.release([root])
    pages.extend(seqs, tails)
    k, v = (torch.cat([t[n][i, :m] for i, m in enumerate(tails)]).contiguous() for n in ("tail_k", "tail_v"))
    torch.cuda.synchronize()
    fill.set(seqs, tails)
    ctx.write_kv_pages_device(fill, 0, kind, k.data_ptr(), width, v.data_ptr(), width)
    pages.extend(seqs, [new] * b)
    s["plan"] = _plan(case, pages, b * new)
    s["plan"].set(seqs, [new] * b)
    ctx.synchronize()


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(state):
    case, t = state["case"], state["t"]
    if not own:
        return {"prompt": _prompt, "batch": _batch, "write": _write, "branch": _branch}[case["op"]](state)
    ctx, pages = state["ctx"], state["pages"]
    if case["op"] == "branch":
        made = pages.fork([state["roots"][p] for p in state["parents"]], [case["length"]] * case["branches"])
        pages.release(state["live"])
        pages.compact()
        state["live"] = made
        tables = np.array([pages.page_ids(q) for q in made], dtype=np.int64)
        return {"pages": state["view"], "tables": tables, "used": pages.used_pages()}
    plan, width = state["plan"], case["kv_heads"] * case["head_dim"]
    source = GGML[case["src"] if case["op"] == "write" else case["q"]]
    ctx.write_kv_pages_device(plan, 0, source, t["k"].data_ptr(), width, t["v"].data_ptr(), width)
    if case["op"] == "write":
        return state["view"]
    wide = case["query_heads"] * case["head_dim"]
    ctx.attention_pages_device(plan, 0, _scale(case), t["q"].data_ptr(), wide, t["o"].data_ptr(), wide)
    return t["o"]


def _softmax(x):
    p = torch.exp(x - x.amax(dim=-1, keepdim=True))
    return p / p.sum(dim=-1, keepdim=True)


def _prompt(state):
    case, t = state["case"], state["t"]
    kvh, hd, n = case["kv_heads"], case["head_dim"], t["q"].shape[0]
    group = case["query_heads"] // kvh
    cached = TYPES[case["kv"]]
    k, v = (t[x].to(cached).float().permute(1, 0, 2).contiguous() for x in ("k", "v"))  # [kvh, n, hd]
    q = t["q"].float().view(n, kvh, group, hd).permute(1, 2, 0, 3).reshape(kvh, group * n, hd)
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * _scale(case)
    back = t["position"][:, None] - t["position"][None, :]
    hidden = (t["sequence"][:, None] != t["sequence"][None, :]) | (back < 0)
    if case["window"]:
        hidden |= back >= case["window"]
    x = x.view(kvh, group, n, n).masked_fill_(hidden, -math.inf).view(kvh, group * n, n)
    o = torch.matmul(_softmax(x), v)
    return o.view(kvh, group, n, hd).permute(2, 0, 1, 3).reshape(n, kvh * group, hd).to(TYPES[case["out"]])


def _batch(state):
    case, t = state["case"], state["t"]
    kvh, hd, b, new, prefix = (case[x] for x in ("kv_heads", "head_dim", "sequences", "new", "prefix"))
    group = case["query_heads"] // kvh
    cached, tail = TYPES[case["kv"]], t["tail_k"].shape[1]
    q = t["q"].float().view(b, new, kvh, group, hd)
    every = q.permute(2, 0, 1, 3, 4).reshape(kvh, b * new * group, hd)
    each = q.permute(0, 2, 1, 3, 4).reshape(b, kvh, new * group, hd)

    def own_part(x):
        return torch.cat([t["tail_" + x], t[x].to(cached)], dim=1).float().permute(0, 2, 1, 3).contiguous()

    def shared_part(x):
        return t["prefix_" + x].float().permute(1, 0, 2).contiguous()

    far = torch.matmul(every, shared_part("k").transpose(1, 2).contiguous())
    far = far.view(kvh, b, new * group, prefix).transpose(0, 1)
    near = torch.matmul(each, own_part("k").transpose(2, 3).contiguous())
    x = (torch.cat([far, near], dim=3) * _scale(case)).view(b, kvh, new, group, prefix + tail + new)
    count = torch.arange(prefix + tail + new, device=x.device)
    fresh = count - (prefix + tail)  # which new token a column is
    length = prefix + t["tails"][:, None]
    at = torch.where(fresh[None, :] >= 0, length + fresh[None, :], count[None, :])  # [b, columns]: positions
    stale = (fresh[None, :] < 0) & (count[None, :] >= length)  # padding behind a shorter tail
    mine = length + torch.arange(new, device=x.device)[None, :]  # [b, new]
    back = mine[:, :, None] - at[:, None, :]
    hidden = stale[:, None, :] | (back < 0)
    if case["window"]:
        hidden = hidden | (back >= case["window"])
    p = _softmax(x.masked_fill(hidden[:, None, :, None, :], -math.inf)).view(b, kvh, new * group, -1)
    p_far = p[..., :prefix].transpose(0, 1).reshape(kvh, b * new * group, prefix)
    o = torch.matmul(p[..., prefix:].contiguous(), own_part("v"))
    o = o + torch.matmul(p_far, shared_part("v")).view(kvh, b, new * group, hd).transpose(0, 1)
    o = o.view(b, kvh, new, group, hd).permute(0, 2, 1, 3, 4).reshape(b, new, kvh * group, hd)
    return o.to(TYPES[case["out"]])


def _write(state):
    """A page holds, for each head, its keys as [dim / 8][64][8] and its values as [8][dim][8], element j of value
    chunk c being token 16 (c / 2) + 4 (c % 2) + 8 (j / 4) + j % 4."""
    t, case = state["t"], state["case"]
    kvh, hd, used = case["kv_heads"], case["head_dim"], state["pages_used"]
    cached, slot, pool = TYPES[case["kv"]], t["slot"], t["pool"]
    chunk = 2 * (slot // 16) + (slot // 4) % 2
    element = 4 * ((slot // 8) % 2) + slot % 4
    pool[:, :, 0].view(used, kvh, hd // 8, PAGE, 8)[t["page"], :, :, slot, :] = t["k"].to(cached).view(-1, kvh, hd // 8, 8)
    pool[:, :, 1].view(used, kvh, PAGE // 8, hd, 8)[t["page"], :, chunk, :, element] = t["v"].to(cached)
    return pool


def _branch(state):
    """The branches' own pages are made behind the live ones and then take the places that the released ones leave."""
    t, case, used = state["t"], state["case"], state["pages_used"]
    pool, n = t["pool"], case["branches"]
    pool[:, used:used + n] = pool[:, t["last"]]
    pool[:, used - n:used] = pool[:, used:used + n]
    shared = case["length"] // PAGE
    tables = torch.cat([t["parents"][:, None] * (shared + 1) + torch.arange(shared, device="cuda")[None, :],
                        torch.arange(used - n, used, device="cuda")[:, None]], dim=1)
    return {"pages": pool[:, :used], "tables": tables, "used": used}


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def _visible(first, count, window):
    """Sum over the positions first .. first + count - 1 of the positions that each sees."""
    return sum(min(p + 1, window or p + 1) for p in range(first, first + count))


def work(case):
    op, kvh, hd = case["op"], case["kv_heads"], case["head_dim"]
    size = {"F32": 4, "F16": 2, "BF16": 2}
    if op == "prompt":
        n, heads = sum(_lengths(case)), case["query_heads"]
        pairs = sum(_visible(0, m, case["window"]) for m in _lengths(case))
        rows = n * hd * (heads * (size[case["q"]] + size[case["out"]]) + 2 * kvh * (size[case["q"]] + 2))
        return {"bytes": rows, "flops": 4.0 * hd * heads * pairs}
    if op == "batch":
        heads, b, new, prefix = case["query_heads"], case["sequences"], case["new"], case["prefix"]
        pairs = sum(_visible(prefix + m, new, case["window"]) for m in _tails(case))
        # cached tokens that any query sees: the prefix's once for all
        starts = [max(0, prefix + m + 1 - case["window"]) if case["window"] else 0 for m in _tails(case)]
        cached = max(0, prefix - min(starts)) + sum(m - max(0, at - prefix) for m, at in zip(_tails(case), starts))
        rows = b * new * hd * (heads * (size[case["q"]] + size[case["out"]]) + 2 * kvh * (size[case["q"]] + 2))
        return {"bytes": rows + cached * 2 * kvh * hd * 2, "flops": 4.0 * hd * heads * pairs}
    if op == "write":
        n = sum(min(m, case["new"] or m) for m in _lengths(case))
        return {"bytes": n * 2 * kvh * hd * (size[case["src"]] + 2), "flops": 0}
    # the cached tokens of a branch's own page are read and written once by the fork and once by the compaction
    own_tokens = case["length"] % PAGE or PAGE
    return {"bytes": 4.0 * case["layers"] * case["branches"] * own_tokens * 2 * kvh * hd * 2, "flops": 0}


# --------------------------------------------------------------------------
# The same in 64 bits
# --------------------------------------------------------------------------
def _one(q, k, v, first, window, scale):
    """One sequence: queries [new, heads, dim] at positions first.. against keys and values [first + new, kvh, dim]."""
    new, heads, hd = q.shape
    n, kvh, _ = k.shape
    o = torch.empty_like(q)
    at = first + torch.arange(new, device=q.device)[:, None] - torch.arange(n, device=q.device)[None, :]
    seen = (at >= 0) & (at < (window or n + new))
    for h in range(heads):
        g = h * kvh // heads
        x = (q[:, h] @ k[:, g].T) * scale
        x[~seen] = -math.inf
        o[:, h] = torch.softmax(x, dim=1) @ v[:, g]
    return o


def exact(case, seed):
    op, hd = case["op"], case["head_dim"]
    t = _inputs(case, seed)
    if op in ("prompt", "batch"):
        cached = TYPES[case["kv"]]
        q = t["q"].double()
        k, v = t["k"].to(cached).double(), t["v"].to(cached).double()
    if op == "prompt":
        o, lo = torch.empty_like(q), 0
        for n in _lengths(case):
            o[lo:lo + n] = _one(q[lo:lo + n], k[lo:lo + n], v[lo:lo + n], 0, case["window"], _scale(case))
            lo += n
        return o
    if op == "batch":
        o = torch.empty_like(q)
        for i, m in enumerate(_tails(case)):
            ks = torch.cat([t["prefix_k"].double(), t["tail_k"][i, :m].double(), k[i]])
            vs = torch.cat([t["prefix_v"].double(), t["tail_v"][i, :m].double(), v[i]])
            o[i] = _one(q[i], ks, vs, case["prefix"] + m, case["window"], _scale(case))
        return o
    if op == "write":
        lengths, kvh = _lengths(case), case["kv_heads"]
        keys = torch.zeros(sum(-(-n // PAGE) for n in lengths), kvh, PAGE, hd, dtype=torch.float64, device="cuda")
        values = torch.zeros_like(keys)
        base = row = 0
        for n in lengths:
            c = min(n, case["new"] or n)
            flat = torch.arange(n - c, n, device="cuda")
            for dst, src in ((keys, t["k"]), (values, t["v"])):
                dst[base + flat // PAGE, :, flat % PAGE] = src[row:row + c].to(TYPES[case["kv"]]).double()
            row, base = row + c, base + -(-n // PAGE)
        ks = keys.view(-1, kvh, PAGE, hd // 8, 8).permute(0, 1, 3, 2, 4).reshape(-1, kvh, 1, hd * PAGE)
        # tokens as (16 s + 8 a + 4 h + i): chunk (s, h), element (a, i)
        vs = values.view(-1, kvh, 4, 2, 2, 4, hd).permute(0, 1, 2, 4, 6, 3, 5).reshape(-1, kvh, 1, hd * PAGE)
        return torch.cat([ks, vs], dim=2)
    last = t["image"].view(case["layers"], case["roots"], -1, t["image"].shape[2])[:, :, -1]
    return {"pages": torch.cat([t["image"], last[:, t["parents"]]], dim=1).double(), "tables": None, "used": None}
