"""Decoding drafted trees and ragged batches over a paged KV cache: what a serving program does between the projections of a step.

Four operators that are used one after another:

* ``plan``       block tables made to fit the requests' lengths, slots, positions and ancestor masks of the new tokens
                 (``gpuk_b200.paged_plan``);
* ``rope``       rotary embedding of queries and keys, and the write of keys and values into their slots (``gpuk_b200.rope_paged``), or of one tensor
                 alone (``gpuk_b200.rope``);
* ``attention``  every new token over its request's pages: single tokens, trees of drafted tokens, prompts (``gpuk_b200.paged_attention``);
* ``keep``       the accepted path of a tree moved to the end of the cached tokens (``gpuk_b200.paged_keep``).

Head counts and sizes are those of the decoders in ``bench.py`` and ``tests/``: 64 / 8, 32 / 8, 16 / 4, 8 / 1 heads of 128, and heads of 64.
``own = False`` computes the operators from elementary PyTorch operations.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _plan(batch, page, ctx, new, tree, **more):
    return dict(kind="plan", batch=batch, page=page, ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1], tree=tree, mix=0, **more)


def _rope(tokens, heads, kv_heads, head_dim, rotary, layout, dtype="bf16", page=16, far=4096, scaling="none", paged=True):
    return dict(kind="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary, layout=layout, dtype=dtype, page=page, far=far,
                scaling=scaling, paged=paged)


def _attention(batch, heads, kv_heads, page, ctx, new, tree, head_dim=128, dtype="bf16", mix=0):
    return dict(kind="attention", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, page=page, ctx_lo=ctx[0], ctx_hi=ctx[1],
                new_lo=new[0], new_hi=new[1], tree=tree, mix=mix)


def _keep(batch, kv_heads, layers, page, ctx, new, head_dim=128, dtype="bf16"):
    return dict(kind="keep", batch=batch, kv_heads=kv_heads, head_dim=head_dim, layers=layers, dtype=dtype, page=page, ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0],
                new_hi=new[1], tree=True, mix=0)


def listed():
    return [
        # a full server that verifies drafts for all its requests
        dict(_plan(256, 16, (1, 4000), (17, 64), True), name="plan trees"),
        # prompts come in: tens of thousands of tokens get positions and slots
        dict(_plan(48, 64, (0, 1000), (1, 3000), False), name="plan prompts"),
        # one token each for a batch of decodes of the large decoder, in the order of pairs that this library's decoder uses
        dict(_rope(32, 64, 8, 128, 128, "split"), name="rope decode"),
        # the new tokens of a prefill
        dict(_rope(8191, 64, 8, 128, 128, "half", page=64), name="rope prompt"),
        # part of the head rotated, positions far beyond the trained context, scaled by parts
        dict(_rope(700, 32, 8, 64, 32, "interleaved", dtype="f16", page=32, far=1000000, scaling="yarn", paged=False), name="rope far partial"),
        # single tokens for a few short requests of the small decoder
        dict(_attention(4, 16, 4, 16, (100, 300), (1, 1), False), name="attention small"),
        # single tokens for a batch of requests of very different lengths
        dict(_attention(32, 64, 8, 64, (30, 4000), (1, 1), False), name="attention ragged"),
        # trees of drafted tokens verified in one pass
        dict(_attention(8, 64, 8, 16, (1500, 2500), (33, 64), True), name="attention trees"),
        # one request with a long context and a tree, heads of 64, fp16
        dict(_attention(1, 32, 8, 32, (30000, 32000), (13, 13), True, head_dim=64, dtype="f16"), name="attention long"),
        # prompts, a continued prompt and single tokens in one batch
        dict(_attention(6, 64, 8, 64, (0, 1984), (2048, 2048), False, mix=4), name="attention prompts"),
        # a few accepted tokens of each request
        dict(_keep(4, 4, 2, 16, (60, 400), (8, 8)), name="keep small"),
        # a full server, several layers at once
        dict(_keep(64, 8, 4, 16, (40, 600), (33, 64)), name="keep many"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "attention", "attention", "keep"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    head_dim = rng.choice([128, 128, 64])
    heads, kv_heads = rng.choice([(64, 8), (32, 8), (16, 4), (8, 1), (16, 16), (24, 8), (28, 4), (5, 5)])
    if kind == "plan":
        tree = rng.random() < 0.6
        lo = _log(rng, 1, 64 if tree else 700)
        hi = _log(rng, lo, 64 if tree else 1500)
        return _plan(_log(rng, 1, 256) if tree else _log(rng, 1, 48), page, (0, _log(rng, 1, 4000)), (lo, hi), tree)
    if kind == "rope":
        rotary = rng.choice([head_dim, head_dim, head_dim // 2, 16])
        return _rope(_log(rng, 1, 8000), heads, kv_heads, head_dim, rotary, rng.choice(["half", "interleaved", "split"]), dtype, page, _log(rng, 100, 1000000),
                     rng.choice(["none", "linear", "base", "bands", "yarn"]), rng.random() < 0.7)
    if kind == "attention":
        form = rng.choice(["token", "tree", "tree", "prompt"])
        batch = _log(rng, 1, {"token": 48, "tree": 12, "prompt": 2}[form])
        top = _log(rng, 20, min(32000, (50000 if form == "token" else 24000) // batch))
        if form == "token":
            return _attention(batch, heads, kv_heads, page, (rng.randint(0, top), top), (1, 1), False, head_dim, dtype)
        if form == "tree":
            return _attention(batch, heads, kv_heads, page, (rng.randint(0, top), top), (rng.randint(1, 8), rng.randint(8, 64)), True, head_dim, dtype)
        new = _log(rng, 2, 1200)
        return _attention(batch, heads, kv_heads, page, (0, rng.choice([0, _log(rng, 1, 1500)])), (rng.randint(1, new), new), False, head_dim, dtype,
                          mix=rng.choice([0, 2]))
    return _keep(_log(rng, 1, 64), rng.choice([1, 4, 8]), rng.randint(1, 4), page, (0, _log(rng, 1, 600)), (rng.randint(2, 8), rng.randint(8, 64)), head_dim, dtype)


# ---- what the requests look like: from the case alone, as `work` needs it ---------------------------------------------
def _lengths(case):
    """Cached and new tokens of each request."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    if case["batch"] > 1 and case["kind"] != "keep":
        ctx[0], ctx[-1] = case["ctx_hi"], case["ctx_lo"]      # the range's ends are there
        new[-1] = case["new_hi"]
    if case["mix"]:      # the first few requests of a prefill batch decode one token
        for i in range(min(case["mix"], case["batch"] - 1)):
            new[i] = 1
    return ctx, new


def _tree(n, rng):
    """Parents of n nodes, each of which comes after its parent: node 0 is the token that was sampled last, the others are drafts behind it."""
    return [-1] + [rng.randint((j - 1) // 4, (j - 1) // 2 if rng.random() < 0.7 else j - 1) for j in range(1, n)]


def _path(parents, rng):
    """A path from the root: the longest of a random leaf's whose moves leave what they read as it is, so that the same pass can be run again."""
    j, path = rng.randrange(len(parents) // 2, len(parents)), []
    while j >= 0:
        path.append(j)
        j = parents[j]
    path.reverse()
    while any(p != i and p < len(path) for i, p in enumerate(path)):
        path.pop()
    return path


def _ceil(a, b):
    return -(-a // b)


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _paged(case, seed, surplus):
    """Pages dealt out to the requests at random: a table whose rows hold the pages of each request's lengths, and the list of the free ones."""
    ctx, new = _lengths(case)
    rng, page = random.Random(seed), case["page"]
    full = [_ceil(c + n, page) for c, n in zip(ctx, new)]
    cached = [_ceil(c, page) for c in ctx]
    width = max(full) + 2
    held = [max(0, min(width, h + (rng.choice([0, 0, 0, 1, 2]) if surplus else 0))) for h in (cached if surplus else full)]
    pages = sum(max(a + 2, b) for a, b in zip(cached, full)) + 7
    order = list(range(pages))
    rng.shuffle(order)
    table = np.full((len(ctx), width), -1, dtype=np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    free = np.zeros(pages, dtype=np.int32)
    free[:pages - at] = order[at:]
    return ctx, new, torch.from_numpy(table).cuda(), held, pages, torch.from_numpy(free).cuda(), pages - at, rng


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _parents(case, new, rng):
    return [_tree(n, rng) for n in new] if case["tree"] else None


def _starts(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def prepare(case, seed):
    s = dict(case)
    if case["kind"] == "rope":
        return _prepare_rope(s, seed)
    ctx, new, table, held, pages, free, count, rng = _paged(case, seed, case["kind"] == "plan")
    s.update(lens=_int(ctx), new=_int(new), tables=table, held=_int(held), pages=pages, free=free, free_count=_int([count, 0]), total=sum(new), longest=max(new),
             most=max(c + n for c, n in zip(ctx, new)))
    s["host"] = list(zip(ctx, new))
    parents = _parents(case, new, rng)
    if parents is not None:
        s["parents"] = _int([p for tree in parents for p in tree])
    if case["kind"] == "plan":
        return s
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    if case["kind"] == "keep":
        s["k"], s["v"] = (_randn(g, case["layers"], *shape).to(dtype) for _ in range(2))
        paths = [_path(p, rng) for p in parents]
        deep = max(map(len, paths)) + 1
        s["paths"] = _int([p + [-1] * (deep - len(p)) for p in paths])
        return s
    s["k"], s["v"] = (_randn(g, *shape).to(dtype) for _ in range(2))
    s["q"] = (_randn(g, s["total"], case["heads"], case["head_dim"]) * 1.5).to(dtype)
    s["starts"] = _int(_starts(new))
    if parents is not None:
        s["masks"] = _int(_mask_words(parents, _ceil(max(new), 32)))
    return s


def _mask_words(parents, words):
    rows = []
    for tree in parents:
        seen = []
        for j, p in enumerate(tree):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        rows += [[((m >> 32 * w & 0xffffffff) ^ 0x80000000) - 0x80000000 for w in range(words)] for m in seen]
    return rows


def _prepare_rope(s, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, t, hd, page = DTYPES[s["dtype"]], s["tokens"], s["head_dim"], s["page"]
    heads, kv = s["heads"], s["kv_heads"]
    rng = random.Random(seed)
    s["positions"] = torch.randint(0, s["far"], (t,), generator=g, device="cuda")
    s["scale"] = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "base": {"kind": "base", "factor": 4.0},
                  "bands": {"kind": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
                  "yarn": {"kind": "yarn", "factor": 16.0, "low": 1.0, "high": 32.0, "original": 4096}}[s["scaling"]]
    if s["paged"]:
        # the projection's output as it lies, queries, keys and values of a token side by side
        qkv = _randn(g, t, heads + 2 * kv, hd).to(dtype)
        s["q"], s["key"], s["value"] = qkv.split([heads, kv, kv], dim=1)
        pages = _ceil(t, page) + 3
        s["slots"] = torch.tensor(rng.sample(range(pages * page), t)).cuda()
        s["k"], s["v"] = (_randn(g, pages, kv, page, hd).to(dtype) for _ in range(2))
    else:
        s["q"] = _randn(g, t, heads, hd).to(dtype)
    if own:
        import gpuk_b200
        s["frequencies"] = gpuk_b200.rope_frequencies(s["rotary"], 500000.0, scaling=s["scale"], device="cuda")
    else:
        f, s["amplitude"] = _frequencies(s["rotary"], 500000.0, s["scale"])
        s["frequencies"] = f.cuda()
    return s


def _frequencies(rotary, theta, scale):
    """Radians a position of each pair, in 64 bits, and the factor of cosines and sines."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64)
    f = theta ** (-i / rotary)
    if scale is None:
        return f, 1.0
    factor = scale["factor"]
    if scale["kind"] == "linear":
        return f / factor, 1.0
    if scale["kind"] == "base":
        return (theta * factor ** (rotary / max(1, rotary - 2))) ** (-i / rotary), 1.0
    turns = scale["original"] * f / (2 * math.pi)      # of a pair over the trained context
    if scale["kind"] == "bands":
        keep = ((turns - scale["low"]) / (scale["high"] - scale["low"])).clamp(0, 1)
        return f / factor * (1 - keep) + f * keep, 1.0
    # yarn: a ramp over the pairs, between those that turn `high` and `low` times
    at = lambda n: rotary * math.log(scale["original"] / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = max(math.floor(at(scale["high"])), 0), min(math.ceil(at(scale["low"])), rotary // 2 - 1)
    ramp = ((i / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import gpuk_b200 as gpuk
    if s["kind"] == "plan":
        p = gpuk.paged_plan(s["lens"], s["new"], s["tables"], s["held"], s["free"], s["free_count"], s["page"], s["total"], parents=s.get("parents"),
                            max_new=s["longest"])
        out = {"starts": p.starts, "positions": p.positions, "slots": p.slots, "held": p.held, "count": p.free_count, "tables": s["tables"], "free": s["free"]}
        if p.masks is not None:
            out["masks"] = p.masks
        return out
    if s["kind"] == "rope":
        if not s["paged"]:
            return gpuk.rope(s["q"], s["positions"], s["frequencies"], layout=s["layout"])
        q = gpuk.rope_paged(s["q"], s["key"], s["value"], s["positions"], s["slots"], s["frequencies"], s["k"], s["v"], layout=s["layout"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if s["kind"] == "attention":
        return gpuk.paged_attention(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["starts"], masks=s.get("masks"), max_len=s["most"])
    return {"lens": gpuk.paged_keep(s["k"], s["v"], s["tables"], s["lens"], s["paths"]), "k": s["k"], "v": s["v"]}


def _run_plain(s):
    return {"plan": _plain_plan, "rope": _plain_rope, "attention": _plain_attention, "keep": _plain_keep}[s["kind"]](s)


def _plain_plan(s):
    page, total, tables, free = s["page"], s["total"], s["tables"], s["free"]
    batch, width = tables.shape
    lens, new, held, count = s["lens"].long(), s["new"].long(), s["held"].long(), s["free_count"][0].long()
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)]).clamp(max=total)
    pages = (lens + new + page - 1) // page
    need = pages.clamp(max=width)
    back, want = (held - need).clamp(min=0), (need - held).clamp(min=0)
    back_at, want_at = back.cumsum(0) - back, want.cumsum(0) - want
    column = torch.arange(width, device=tables.device)[None]
    # pages that are too many go on top of the list, those that are missing come from its top
    given = (column >= need[:, None]) & (column < held[:, None])
    to = torch.where(given, count + back_at[:, None] + column - need[:, None], free.numel())
    free = torch.cat([free, free.new_zeros(1)]).scatter(0, to.view(-1), tables.view(-1))[:-1]
    there = count + back.sum()
    taken = (column >= held[:, None]) & (column < need[:, None])
    at = there - 1 - (want_at[:, None] + column - held[:, None])
    tables = torch.where(taken, torch.where(at >= 0, free[at.clamp(0, free.numel() - 1)], -1), tables)
    got = torch.minimum(want, (there - want_at).clamp(min=0))
    left = (there - want.sum()).clamp(min=0)
    missing = want.sum() - (there - left) + (pages - need).sum()
    t = torch.arange(total, device=tables.device)
    request = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    index = t - starts[request]
    at = lens[request] + index
    block = tables[request, (at // page).clamp(max=width - 1)].long()
    slots = torch.where((at // page < width) & (block >= 0), block * page + at % page, -1)
    out = {"starts": starts.int(), "slots": slots, "held": (held - back + got).int(), "count": torch.stack([left, missing]).int(), "tables": tables, "free": free}
    if "parents" not in s:
        return dict(out, positions=at)
    # a node's ancestors and itself, by squaring the relation
    n = s["longest"]
    parent = s["parents"].long()
    above = torch.zeros(batch, n, n, device=tables.device)
    above[request, index, index] = 1
    rows = torch.where(parent >= 0, request * n * n + index * n + parent, (request * n + index) * n + index)
    above.view(-1).index_fill_(0, rows, 1)
    for _ in range(max(1, (n - 1).bit_length())):
        above = (above @ above > 0).float()
    seen = above[request, index]
    words = _ceil(n, 32)
    bits = torch.nn.functional.pad(seen, (0, words * 32 - n)).long().view(total, words, 32)
    masks = (bits << torch.arange(32, device=tables.device)).sum(-1).to(torch.int32)
    return dict(out, positions=lens[request] + seen.sum(-1).long() - 1, masks=masks)


def _plain_rotate(s, x):
    """The first `rotary` values of each head rotated by the token's angles, in 32 bits, from angles in 64."""
    r, layout = s["rotary"], s["layout"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    x = x.float()
    part = x[..., :r]
    a, b = (part[..., :r // 2], part[..., r // 2:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([lo, hi], -1).flatten(-2) if layout == "interleaved" else torch.cat([lo, hi], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_rope(s):
    q = _plain_rotate(s, s["q"]).to(s["q"].dtype)
    if not s["paged"]:
        return q
    page = s["page"]
    block, at = s["slots"] // page, s["slots"] % page
    s["k"][block, :, at] = _plain_rotate(s, s["key"]).to(q.dtype)
    s["v"][block, :, at] = s["value"]
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    """All requests at once where the scores of the padded batch are few, else one after another."""
    sizes, heads, kv, hd = s["host"], s["heads"], s["kv_heads"], s["head_dim"]
    most, longest = s["most"], s["longest"]
    q, masks = s["q"], s.get("masks")
    if len(sizes) * heads * longest * most <= 1 << 28:
        t = torch.arange(s["total"], device=q.device)
        request = torch.searchsorted(s["starts"][1:].contiguous(), t, right=True)
        index = t - s["starts"][request]
        padded = q.new_zeros(len(sizes), longest, heads, hd, dtype=torch.float32)
        padded[request, index] = q.float()
        bits = None
        if masks is not None:
            bits = masks.new_zeros(len(sizes), longest, masks.shape[1])
            bits[request, index] = masks
        return _attend(s, padded, s["tables"], s["lens"], s["new"], bits, most)[request, index].to(q.dtype)
    out, at = [], 0
    for i, (c, n) in enumerate(sizes):
        rows = slice(at, at + n)
        out.append(_attend(s, q[rows].float()[None], s["tables"][i:i + 1], s["lens"][i:i + 1], s["new"][i:i + 1], None if masks is None else masks[rows][None], c + n)[0])
        at += n
    return torch.cat(out).to(q.dtype)


def _attend(s, q, tables, lens, new, bits, most):
    batch, n, heads, hd = q.shape
    kv, page = s["kv_heads"], s["page"]
    used = tables[:, :_ceil(most, page)].long().clamp(min=0)
    k, v = (c[used].permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, hd)[:, :, :most].float() for c in (s["k"], s["v"]))
    key = torch.arange(most, device=q.device)[None, None]
    row = torch.arange(n, device=q.device)[None, :, None]
    behind = key - lens[:, None, None]      # which of the new tokens a key is
    if bits is None:
        seen = behind <= row
    else:
        word = bits.gather(2, (behind.clamp(0, n - 1) >> 5).expand(batch, n, most).long())
        seen = (behind < 0) | ((word >> (behind.clamp(min=0) & 31) & 1) == 1)
    seen = (seen & (behind < new[:, None, None]))[:, None, :, None]
    scores = torch.einsum("bnghd,bgld->bgnhl", q.view(batch, n, kv, heads // kv, hd), k) / math.sqrt(hd)
    scores = scores.masked_fill(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bgnhl,bgld->bgnhd", p, v) / torch.where(total == 0, 1, total)
    return o.permute(0, 2, 1, 3, 4).reshape(batch, n, heads, hd)


def _plain_keep(s):
    page, paths = s["page"], s["paths"].long()
    deep = paths.shape[1]
    good = paths >= 0
    rows = torch.arange(paths.shape[0], device=paths.device)[:, None]
    source = s["lens"].long()[:, None] + paths.clamp(min=0)
    target = s["lens"].long()[:, None] + torch.arange(deep, device=paths.device)
    target = torch.where(good, target, source[:, :1])      # what is no move takes the first token to where it is
    source = torch.where(good, source, source[:, :1])
    src, dst = s["tables"][rows, source // page].long(), s["tables"][rows, target // page].long()
    for cache in (s["k"], s["v"]):
        cache[:, dst, :, target % page] = cache[:, src, :, source % page]
    return {"lens": (s["lens"] + good.sum(1)).int(), "k": s["k"], "v": s["v"]}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "rope":
        row = case["head_dim"] * 2
        heads = case["heads"] + (2 * case["kv_heads"] if case["paged"] else 0)
        turned = case["heads"] + (case["kv_heads"] if case["paged"] else 0)
        return {"bytes": case["tokens"] * (2 * heads * row + (16 if case["paged"] else 8)), "flops": case["tokens"] * turned * case["rotary"] * 3}
    ctx, new = _lengths(case)
    batch, total, page = case["batch"], sum(new), case["page"]
    if case["kind"] == "plan":
        words = _ceil(max(new), 32) if case["tree"] else 0
        fresh = sum(_ceil(c + n, page) - _ceil(c, page) for c, n in zip(ctx, new))
        return {"bytes": total * (16 + 4 * words + (4 if case["tree"] else 0)) + batch * 20 + fresh * 8, "flops": total * 4}
    row = case["head_dim"] * 2
    if case["kind"] == "keep":
        moved = sum(len(p) for p in (_path(_tree(n, r), r) for n, r in ((n, random.Random(i)) for i, n in enumerate(new))))
        return {"bytes": 4 * moved * case["layers"] * case["kv_heads"] * row + batch * 8, "flops": 0}
    # keys that a request's tokens see: the cached ones, and of the new ones those up to itself, or in a tree about as many as a balanced one is deep
    pairs = sum(n * c + (n * (n + 1) // 2 if not case["tree"] else n * n.bit_length()) for c, n in zip(ctx, new))
    cached = sum(c + n for c, n in zip(ctx, new))
    return {"bytes": 2 * cached * case["kv_heads"] * row + 2 * total * case["heads"] * row + 4 * _ceil(cached, page),
            "flops": 4 * case["head_dim"] * case["heads"] * pairs}


# ---- the operators' definitions in 64 bits -------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"plan": _exact_plan, "rope": _exact_rope, "attention": _exact_attention, "keep": _exact_keep}[case["kind"]](case, s)


def _exact_plan(case, s):
    page, total = case["page"], s["total"]
    lens, new, held, tables, free = (s[k].cpu().tolist() for k in ("lens", "new", "held", "tables", "free"))
    count, _ = s["free_count"].tolist()
    width, missing = len(tables[0]), 0
    want = [min(_ceil(c + n, page), width) for c, n in zip(lens, new)]
    for i, w in enumerate(want):
        for j in range(w, held[i]):
            free[count] = tables[i][j]
            count += 1
    out_held = []
    for i, w in enumerate(want):
        have = min(held[i], w)
        for j in range(held[i], w):
            if count:
                count -= 1
                tables[i][j] = free[count]
                have += 1
            else:
                tables[i][j] = -1
                missing += 1
        missing += _ceil(lens[i] + new[i], page) - w
        out_held.append(have)
    parents = s["parents"].tolist() if "parents" in s else None
    positions, slots, masks, starts = [], [], [], [0]
    for i, (c, n) in enumerate(zip(lens, new)):
        depth, seen = [], []
        for j in range(n):
            block = (c + j) // page
            there = block < width and tables[i][block] >= 0
            slots.append(tables[i][block] * page + (c + j) % page if there else -1)
            if parents is None:
                positions.append(c + j)
                continue
            p = parents[starts[-1] + j]
            depth.append(depth[p] + 1 if p >= 0 else 0)
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
            positions.append(c + depth[-1])
        masks += seen
        starts.append(starts[-1] + n)
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t)  # noqa: E731
    out = {"starts": ints(starts), "positions": ints(positions, torch.int64), "slots": ints(slots, torch.int64), "held": ints(out_held), "count": ints([count, missing]),
           "tables": ints(tables), "free": ints(free)}
    if parents is not None:
        words = _ceil(max(new), 32)
        out["masks"] = ints([[((m >> 32 * w & 0xffffffff) ^ 0x80000000) - 0x80000000 for w in range(words)] for m in masks])
    return out


def _exact_rope(case, s):
    r, half = case["rotary"], case["rotary"] // 2
    f, amplitude = _frequencies(r, 500000.0, s["scale"])
    # whole turns are taken out of the angle before it is one: far positions lose nothing
    turns = torch.remainder(s["positions"].double()[:, None] * (f / (2 * math.pi)).cuda(), 1.0)
    turn = torch.polar(torch.full_like(turns, amplitude), 2 * math.pi * turns)[:, None]

    def rotated(x):
        x = x.double()
        first = list(range(half)) if case["layout"] == "half" else list(range(0, r, 2))
        second = [i + half for i in first] if case["layout"] == "half" else [i + 1 for i in first]
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        if case["layout"] == "split":
            first, second = list(range(half)), list(range(half, r))
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if not case["paged"]:
        return rotated(s["q"])
    k, v = s["k"].double(), s["v"].double()
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    k.view(-1, *k.shape[2:])[s["slots"]] = rotated(s["key"])
    v.view(-1, *v.shape[2:])[s["slots"]] = s["value"].double()
    return {"q": rotated(s["q"]), "k": k.transpose(1, 2), "v": v.transpose(1, 2)}


def _exact_attention(case, s):
    page, hd, group = case["page"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (c, n) in enumerate(s["host"]):
        place = torch.arange(c + n, device="cuda")
        block, inside = s["tables"][i].long()[place // page], place % page
        seen = torch.ones(n, c + n, dtype=torch.bool, device="cuda")
        if "masks" in s:
            word = s["masks"][at:at + n].long() & 0xffffffff
            j = torch.arange(n, device="cuda")
            seen[:, c:] = (word[:, j // 32] >> (j % 32) & 1).bool()
        else:
            seen = seen.tril(c)
        for h in range(case["kv_heads"]):
            k, v = s["k"][block, h, inside].double(), s["v"][block, h, inside].double()
            for g in range(group):
                score = s["q"][at:at + n, h * group + g].double() @ k.T / math.sqrt(hd)
                out[at:at + n, h * group + g] = torch.softmax(torch.where(seen, score, -math.inf), -1) @ v
        at += n
    return out


def _exact_keep(case, s):
    page, lens, paths, tables = case["page"], s["lens"].tolist(), s["paths"].tolist(), s["tables"].tolist()
    k, v = s["k"].double(), s["v"].double()
    after = []
    for i, path in enumerate(paths):
        path = [p for p in path if p >= 0]
        for j, p in enumerate(path):
            a, b = lens[i] + p, lens[i] + j
            for cache in (k, v):
                cache[:, tables[i][b // page], :, b % page] = cache[:, tables[i][a // page], :, a % page]
        after.append(lens[i] + len(path))
    return {"lens": torch.tensor(after, dtype=torch.int32), "k": k, "v": v}
