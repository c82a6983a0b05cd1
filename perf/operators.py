"""The operators of a cache in pages whose speed counts: attention of drafted tokens over the pages, and what moves and
hands out the pages themselves. `listed()` names some calls, `draw()` gives more of the same ranges, `run()` makes one in
its plain form (elementary torch operations in 32 bits) or, where `own` is true, through `ytensor_b200.paged`, and
`exact()` says what comes out in 64 bits.

A pool holds the keys and values of all layers in pages, [layers, pages, key/value heads, positions of a page, dim]. A slot
is one sequence: `lens` positions, in the pages that its row of `table` names (`held` of them); `refs` counts the slots that
hold a page. Kinds of case:
  attend   rows of drafted tokens (a tree by its parents, or a plain chain) are stored behind their sequences and attend to
           the sequence and to their own ancestors, in one layer
  append   rows of new tokens are stored behind their sequences, in one layer
  keep     of the drafted rows the accepted ones move together, in every layer, and the lengths grow
  fork     slots become copies of others (beam search), then make room to be written: pages that others hold too are copied
  compact  the pages in use go to the front of another pool
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one user, one token at a time: what a call costs at the least
        {"name": "attend_one", "kind": "attend", "slots": 1, "context": 1000, "nodes": 1, "tree": False, "kv": 8, "groups": 2,
         "dim": 128, "page": 16, "dtype": "bf16", "layers": 2},
        # many users, one token each, long and ragged contexts
        {"name": "attend_many", "kind": "attend", "slots": 32, "context": 16384, "nodes": 1, "tree": False, "kv": 8,
         "groups": 4, "dim": 128, "page": 16, "dtype": "bf16", "layers": 1},
        # small trees in the default number format, odd lengths
        {"name": "attend_tree_f32", "kind": "attend", "slots": 4, "context": 2001, "nodes": 13, "tree": True, "kv": 8,
         "groups": 2, "dim": 128, "page": 16, "dtype": "f32", "layers": 2},
        # wide trees of several users over long contexts: products of hundreds of rows
        {"name": "attend_tree_wide", "kind": "attend", "slots": 8, "context": 16000, "nodes": 64, "tree": True, "kv": 8,
         "groups": 4, "dim": 128, "page": 32, "dtype": "f16", "layers": 1},
        # the rows of a few drafted tokens
        {"name": "append_tree", "kind": "append", "slots": 16, "context": 1000, "nodes": 24, "kv": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "layers": 2},
        # the rows of whole prompts
        {"name": "append_prompts", "kind": "append", "slots": 4, "context": 0, "nodes": 8000, "kv": 8, "dim": 128, "page": 64,
         "dtype": "f32", "layers": 1},
        # one user's accepted tokens in a model of 28 layers
        {"name": "keep_one", "kind": "keep", "slots": 1, "context": 700, "nodes": 24, "kept": 5, "kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "layers": 28},
        # many users' accepted tokens
        {"name": "keep_many", "kind": "keep", "slots": 64, "context": 800, "nodes": 48, "kept": 12, "kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "layers": 28},
        # a beam search of four beams
        {"name": "fork_beams", "kind": "fork", "slots": 4, "beams": 4, "context": 1003, "nodes": 1, "kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "layers": 28},
        # several beam searches behind long prompts, large pages
        {"name": "fork_many", "kind": "fork", "slots": 64, "beams": 8, "context": 8100, "nodes": 16, "kv": 4, "dim": 128,
         "page": 64, "dtype": "f16", "layers": 12},
        # a small pool, half of it in use
        {"name": "compact_small", "kind": "compact", "slots": 8, "beams": 2, "context": 500, "kv": 4, "dim": 64, "page": 16,
         "dtype": "bf16", "layers": 4},
        # a pool of more than a gigabyte
        {"name": "compact_pool", "kind": "compact", "slots": 48, "beams": 4, "context": 5000, "kv": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "layers": 8},
    ]


# ---------------------------------------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    """A whole number, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["attend"] * 4 + ["append", "keep", "fork", "compact"])
        c = {"kind": kind, "slots": _log(rng, 1, 64), "context": _log(rng, 1, 20000), "kv": rng.choice([1, 2, 4, 8]),
             "dim": rng.choice([64, 80, 128, 128, 128, 256]), "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128]),
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "layers": rng.choice([1, 2])}
        if kind == "attend":
            c["groups"] = rng.choice([1, 2, 3, 4, 8])
            c["nodes"] = rng.choice([1, _log(rng, 2, 128)])
            c["tree"] = c["nodes"] > 1 and rng.random() < 0.7
        elif kind == "append":
            c["nodes"] = _log(rng, 1, 8000)
        else:
            c["layers"] = rng.choice([4, 12, 28])
        if kind == "keep":
            c["nodes"] = _log(rng, 1, 64)
            c["kept"] = rng.randint(1, min(16, c["nodes"]))
        elif kind in ("fork", "compact"):
            c["beams"] = rng.choice([1, 2, 4, 8])
            if kind == "fork":
                c["nodes"] = rng.choice([1, 16])
        w = work(c)
        pool = 1.3 * _pool_pages(c) * c["page"] * c["layers"] * c["kv"] * 2 * c["dim"] * SIZE[c["dtype"]]
        if pool < 4e9 and w["bytes"] < 1.3e9 and w["flops"] < (1e11 if c["dtype"] != "f32" else 5e9):
            return c


# ---------------------------------------------------------------------------------------------- sizes
def _sizes(c):
    """(lengths, new tokens) of the slots: ragged, the first slot as long as the case says, the last of many idle."""
    rng = random.Random("%d %d %d" % (c["slots"], c["context"], c.get("nodes", 0)))
    lens = [c["context"]] + [rng.randint(c["context"] // 4, c["context"]) for _ in range(c["slots"] - 1)]
    n = c.get("nodes", 0)
    nodes = [n] + [rng.randint(1, n) if n else 0 for _ in range(c["slots"] - 1)]
    if c["slots"] > 4 and c["kind"] in ("attend", "append"):
        nodes[-1] = 0
    if "beams" in c:  # the beams of one search are equally long
        lens = [lens[s // c["beams"] * c["beams"]] for s in range(c["slots"])]
    return lens, nodes


def _shared(c, s, length):
    """How many of slot s's first pages it holds together with the first slot of its beams."""
    return length // c["page"] if s % c.get("beams", 1) else 0


def _pool_pages(c):
    lens, nodes = _sizes(c)
    return sum(-(-(l + n) // c["page"]) - _shared(c, s, l) for s, (l, n) in enumerate(zip(lens, nodes)))


def _sources(c):
    """For each slot the beam of its own search that it goes on from."""
    rng = random.Random("%d %d" % (c["slots"], c["context"]))
    b, n = c["beams"], c["slots"]
    return [min(n - 1, s // b * b + rng.randrange(b)) for s in range(n)]


def work(case):
    c = case
    lens, nodes = _sizes(c)
    row = c["kv"] * c["dim"] * SIZE[c["dtype"]]  # the keys of one position in one layer
    total = sum(nodes)
    if c["kind"] == "attend":
        heads = c["kv"] * c["groups"]
        seen = sum(l for l, n in zip(lens, nodes) if n)
        pairs = sum(n * (l + 1) for l, n in zip(lens, nodes))
        return {"bytes": 2 * row * (seen + 2 * total) + 2 * total * row * c["groups"], "flops": 4 * pairs * heads * c["dim"]}
    if c["kind"] == "append":
        return {"bytes": 4 * row * total, "flops": 0}
    if c["kind"] == "keep":  # (the first accepted row of a tree is where it was)
        return {"bytes": 4 * row * c["layers"] * sum(k - 1 for k in _kept(c)) + 12 * c["slots"], "flops": 0}
    table = 4 * sum(-(-l // c["page"]) for l in lens)
    if c["kind"] == "fork":
        src = _sources(c)
        copied = sum(lens[s] % c["page"] for s in range(c["slots"]) if src.count(src[s]) > 1)
        return {"bytes": 4 * row * c["layers"] * copied + 2 * table, "flops": 0}
    return {"bytes": 4 * row * c["layers"] * c["page"] * _pool_pages(c) + 2 * table, "flops": 0}


def _kept(c):
    rng = random.Random("%d %d" % (c["slots"], c["kept"]))
    return [min(n, rng.randint(1, c["kept"])) for n in _sizes(c)[1]]


# ---------------------------------------------------------------------------------------------- inputs
def _pool(c, g, pages):
    shape = (c["layers"], pages, c["kv"], c["page"], c["dim"])
    return torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[c["dtype"]])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def prepare(case, seed):
    c, rng = case, random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    lens, nodes = _sizes(c)
    slots, page = c["slots"], c["page"]
    # pages lie anywhere in the pool; a fifth of it and room to copy pages is free
    used = _pool_pages(c)
    pages = used + used // 5 + 2 * slots * (1 + c.get("nodes", 0) // page)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))[:used].tolist()
    if c["kind"] == "compact":  # two pages in three are free
        order = torch.randperm(3 * used, generator=torch.Generator().manual_seed(int(seed)))[:used].tolist()
        pages = 3 * used
    # a fork makes room itself: its slots hold no more than their positions
    ends = lens if c["kind"] in ("fork", "compact") else [l + n for l, n in zip(lens, nodes)]
    max_pages = max(-(-(l + n) // page) for l, n in zip(lens, nodes)) + 1
    table, held, refs = torch.full((slots, max_pages), -1, dtype=torch.int32), [], torch.zeros(pages, dtype=torch.int32)
    at = 0
    for s in range(slots):
        n, m = -(-ends[s] // page), _shared(c, s, lens[s])
        first = s // c.get("beams", 1) * c.get("beams", 1)
        table[s, :m] = table[first, :m]
        table[s, m:n] = torch.tensor(order[at:at + n - m], dtype=torch.int32)
        at += n - m
        held.append(n)
        refs[table[s, :n].long()] += 1
    st = {"case": c, "k": _pool(c, g, pages), "v": _pool(c, g, pages), "table": table.cuda(), "refs": refs.cuda(),
          "lens": _ints(lens), "held": _ints(held), "longest": max(lens), "most": max(nodes)}
    dt, total = DTYPES[c["dtype"]], sum(nodes)
    if c["kind"] in ("attend", "append"):
        st["starts"] = _ints([sum(nodes[:s]) for s in range(slots + 1)])
        st["k_new"], st["v_new"] = (torch.randn((total, c["kv"], c["dim"]), generator=g, device="cuda", dtype=dt)
                                    for _ in range(2))
    if c["kind"] == "attend":
        st["q"] = torch.randn((total, c["kv"] * c["groups"], c["dim"]), generator=g, device="cuda", dtype=dt)
        # a node hangs on one of the few before it, the first on the sequence
        st["parents"] = _ints([max(-1, i - 1 - rng.randrange(6)) for n in nodes for i in range(n)]) if c["tree"] else None
    elif c["kind"] == "keep":
        st["kept"] = _ints(_kept(c))
        st["accepted"] = torch.zeros(slots, c["kept"], dtype=torch.int32)
        for s, k in enumerate(_kept(c)):
            st["accepted"][s, :k] = torch.tensor([0] + sorted(rng.sample(range(1, nodes[s]), k - 1)), dtype=torch.int32)
        st["accepted"], st["base"] = st["accepted"].cuda(), st["lens"].clone()
    elif c["kind"] == "fork":
        st["source"], st["counts"] = _ints(_sources(c)), _ints(nodes)
    elif c["kind"] == "compact":
        small = used + used // 8
        st["into"] = {"k": torch.zeros_like(st["k"][:, :small]), "v": torch.zeros_like(st["v"][:, :small]),
                      "table": torch.full_like(st["table"], -1), "refs": torch.zeros_like(st["refs"][:small]),
                      "lens": torch.zeros_like(st["lens"]), "held": torch.zeros_like(st["held"])}
    if own:  # the handle that a program keeps over its pools
        from ytensor_b200.paged import PagedCache
        for t in [st] + ([st["into"]] if "into" in st else []):
            t["cache"] = PagedCache.over(t["k"], t["v"], t["table"], t["lens"], t["held"], t["refs"])
    return st


# ---------------------------------------------------------------------------------------------- a pass
def _pages_of(s):
    return {n: s[n] for n in ("k", "v", "table", "lens", "held", "refs")}


def run(state):
    c, s = state["case"], state
    kind, layer = c["kind"], c["layers"] - 1
    if own:
        cache = s["cache"]
        if kind == "attend":
            out = cache.attend(layer, s["q"], s["starts"], s["k_new"], s["v_new"], parents=s["parents"])
            return {"out": out, "k": s["k"], "v": s["v"]}
        if kind == "append":
            cache.append(layer, s["k_new"], s["v_new"], s["starts"])
            return {"k": s["k"], "v": s["v"]}
        if kind == "keep":
            cache.keep(s["kept"], s["accepted"], base=s["base"])
            return _pages_of(s)
        if kind == "fork":
            cache.fork(s["source"])
            cache.reserve(s["counts"])
            return _pages_of(s)
        cache.compact(s["into"]["cache"])
        return _pages_of(s["into"])
    if kind == "attend":
        _append(s, layer)
        return {"out": _attend(s, layer), "k": s["k"], "v": s["v"]}
    if kind == "append":
        _append(s, layer)
        return {"k": s["k"], "v": s["v"]}
    if kind == "keep":
        _keep(s)
        return _pages_of(s)
    if kind == "fork":
        _fork(s)
        _reserve(s)
        return _pages_of(s)
    _compact(s, s["into"])
    return _pages_of(s["into"])


# ---------------------------------------------------------------------------------------------- the plain form
def _places(s, positions):
    """Pages and rows of positions [slots, n]."""
    page = s["case"]["page"]
    at = (positions // page).clamp(max=s["table"].shape[1] - 1)
    return s["table"].gather(1, at).long().clamp(min=0), positions % page


def _append(s, layer):
    starts = s["starts"].long()
    rows = torch.arange(s["k_new"].shape[0], device="cuda")
    slot = torch.searchsorted(starts, rows, right=True) - 1
    position = s["lens"].long()[slot] + rows - starts[slot]
    page = s["table"][slot, position // s["case"]["page"]].long()
    for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        pool[layer][page, :, position % s["case"]["page"]] = new


def _ancestors(parents, starts, most):
    """[slots, most, most]: whether node j is i or an ancestor of it."""
    n = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=parents.numel() - 1)
    up = torch.where(i < n[:, None], parents.long()[row], -1)
    seen = ((up[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (most - 1).bit_length())):  # paths of twice the length
        seen = (seen @ seen).clamp(max=1)
    return seen > 0


def _attend(s, layer):
    c = s["case"]
    starts, lens, most, slots = s["starts"].long(), s["lens"].long(), s["most"], c["slots"]
    n = starts[1:] - starts[:-1]
    page, row = _places(s, torch.arange(s["longest"] + most, device="cuda").expand(slots, -1))
    k, v = (pool[layer][page, :, row].float() for pool in (s["k"], s["v"]))  # [slots, positions, heads, dim]
    i = torch.arange(most, device="cuda")
    at = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().reshape(slots, most, c["kv"], c["groups"], c["dim"])
    scores = torch.einsum("sihgd,slhd->shgil", q, k) * c["dim"] ** -0.5
    j = torch.arange(k.shape[1], device="cuda") - lens[:, None]  # the node at a position; negative: the sequence itself
    if s["parents"] is not None:
        own_path = _ancestors(s["parents"], starts, most).gather(2, j.clamp(0, most - 1)[:, None].expand(-1, most, -1))
    else:
        own_path = j[:, None] <= i[:, None]
    seen = (j < 0)[:, None] | (own_path & (j < n[:, None])[:, None])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    # (behind a sequence's end lie other sequences' rows: weights of zero)
    out = torch.einsum("shgil,slhd->sihgd", p, v).reshape(slots, most, -1, c["dim"])
    return out[i < n[:, None]].to(s["q"].dtype)


def _keep(s):
    page, depth = s["case"]["page"], s["accepted"].shape[1]
    j = torch.arange(depth, device="cuda")
    slot, place = torch.nonzero(j < s["kept"][:, None], as_tuple=True)
    base = s["base"].long()[slot]
    source, target = base + s["accepted"][slot, place], base + place
    a, b = (s["table"][slot, p // page].long() for p in (source, target))
    for pool in (s["k"], s["v"]):
        rows = pool.permute(1, 3, 0, 2, 4)  # [pages, rows, layers, heads, dim]
        rows[b, target % page] = rows[a, source % page]
    s["lens"].copy_(s["base"] + s["kept"])


def _fork(s):
    page, src, slots = s["case"]["page"], s["source"].long(), s["case"]["slots"]
    moves, gone = src != torch.arange(slots, device="cuda"), src < 0
    src = src.clamp(min=0)
    lens = torch.where(gone, 0, s["lens"][src])
    held = torch.where(moves, (lens + page - 1) // page, s["held"])
    at = torch.arange(s["table"].shape[1], device="cuda")
    before, behind = at < s["held"][:, None], at < held[:, None]
    table = torch.where(moves[:, None] & behind, s["table"][src], s["table"])
    change = torch.zeros_like(s["refs"])
    for rows, which, by in ((s["table"], before, -1), (table, behind, 1)):
        ids = rows[which & moves[:, None]].long()
        change.index_add_(0, ids, torch.full_like(ids, by, dtype=torch.int32))
    s["refs"] += change
    s["table"].copy_(table)
    s["lens"].copy_(torch.where(moves, lens, s["lens"]))
    s["held"].copy_(held)


def _reserve(s):
    page, slots = s["case"]["page"], s["case"]["slots"]
    lens, held, counts = s["lens"].long(), s["held"].long(), s["counts"].long()
    last = lens // page
    at = s["table"].gather(1, last.clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0].long()
    copy = (counts > 0) & (lens % page > 0) & (s["refs"][at.clamp(min=0)] > 1)
    need = torch.where(counts > 0, (lens + counts + page - 1) // page, 0)
    want = (need - held).clamp(min=0) + copy
    free = torch.nonzero(s["refs"] == 0)[:, 0]
    total = int(want.sum())
    if total > free.numel() or int(need.max()) > s["table"].shape[1]:
        return
    fresh = free[:total]
    before = want.cumsum(0) - want
    slot = torch.repeat_interleave(torch.arange(slots, device="cuda"), want)
    r = torch.arange(total, device="cuda") - before[slot]
    first = copy[slot] & (r == 0)
    s["table"][slot, torch.where(first, last[slot], held[slot] + r - copy[slot].long())] = fresh.to(torch.int32)
    s["refs"][fresh] = 1
    s["refs"].index_add_(0, at[copy], torch.full_like(at[copy], -1, dtype=torch.int32))
    s["held"].copy_(torch.maximum(held, need))
    target = fresh[before[copy]]
    filled = (torch.arange(page, device="cuda") < (lens % page)[copy][:, None])[None, :, None, :, None]
    for pool in (s["k"], s["v"]):
        pool[:, target] = torch.where(filled, pool[:, at[copy]], pool[:, target])


def _compact(s, into):
    live = s["refs"] > 0
    ids = torch.nonzero(live)[:, 0]
    number = (live.cumsum(0) - 1).to(torch.int32)
    holds = torch.arange(s["table"].shape[1], device="cuda") < s["held"][:, None]
    into["table"].copy_(torch.where(holds, number[s["table"].long().clamp(min=0)], into["table"]))
    into["lens"].copy_(s["lens"])
    into["held"].copy_(s["held"])
    into["refs"].zero_()
    into["refs"][:ids.numel()] = s["refs"][ids]
    for n in ("k", "v"):
        into[n][:, :ids.numel()] = s[n][:, ids]


# ---------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """Slot by slot and page by page, from what the operators are said to do."""
    c = case
    s = prepare(c, seed)
    page, layer = c["page"], c["layers"] - 1
    table, lens, held, refs = ([list(r) if isinstance(r, list) else r for r in s[n].tolist()]
                               for n in ("table", "lens", "held", "refs"))
    if c["kind"] in ("attend", "append"):
        starts = s["starts"].tolist()
        if starts[-1] // page > 50000:  # (too many steps)
            return None
        for b in range(c["slots"]):
            done = 0
            while done < starts[b + 1] - starts[b]:  # as many rows as the page still takes
                at = lens[b] + done
                n = min(page - at % page, starts[b + 1] - starts[b] - done)
                for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
                    pool[layer, table[b][at // page], :, at % page:at % page + n] = \
                        new[starts[b] + done:starts[b] + done + n].transpose(0, 1)
                done += n
        got = {"k": s["k"], "v": s["v"]}
        if c["kind"] == "attend":
            got["out"] = _exact_attention(c, s, layer, table, lens, starts)
        return got
    if c["kind"] == "keep":
        kept, accepted, base = s["kept"].tolist(), s["accepted"].tolist(), s["base"].tolist()
        for b in range(c["slots"]):
            for to, i in enumerate(accepted[b][:kept[b]]):
                x, y = base[b] + i, base[b] + to
                for pool in (s["k"], s["v"]):
                    pool[:, table[b][y // page], :, y % page] = pool[:, table[b][x // page], :, x % page].clone()
            s["lens"][b] = base[b] + kept[b]
        return _pages_of(s)
    if c["kind"] == "fork":
        source, counts = s["source"].tolist(), s["counts"].tolist()
        old = [row[:h] for row, h in zip(table, held)]
        for b, a in enumerate(source):
            if a != b:
                held[b] = -(-lens[a] // page)
                table[b][:held[b]] = old[a][:held[b]]
        lens = [lens[a] for a in source]
        refs = _counted(table, held, len(refs))
        free, shared = iter([p for p, r in enumerate(refs) if not r]), list(refs)
        for b in range(c["slots"]):
            last = lens[b] // page
            if lens[b] % page and shared[table[b][last]] > 1:
                new = next(free)
                for pool in (s["k"], s["v"]):
                    pool[:, new, :, :lens[b] % page] = pool[:, table[b][last], :, :lens[b] % page].clone()
                table[b][last] = new
            while held[b] < -(-(lens[b] + counts[b]) // page):
                table[b][held[b]] = next(free)
                held[b] += 1
        return {"k": s["k"], "v": s["v"], "table": _ints(table), "lens": _ints(lens), "held": _ints(held),
                "refs": _ints(_counted(table, held, len(refs)))}
    into, number = s["into"], {}
    for p in [p for p, r in enumerate(refs) if r]:
        number[p] = len(number)
    for pool in ("k", "v"):
        for a in range(0, c["layers"]):
            into[pool][a, :len(number)] = torch.index_select(s[pool][a], 0, torch.tensor(list(number), device="cuda"))
    out = [[number[p] if i < held[b] else -1 for i, p in enumerate(row)] for b, row in enumerate(table)]
    return {"k": into["k"], "v": into["v"], "table": _ints(out), "lens": s["lens"], "held": s["held"],
            "refs": _ints([refs[p] for p in number] + [0] * (into["refs"].numel() - len(number)))}


def _counted(table, held, pages):
    refs = [0] * pages
    for row, h in zip(table, held):
        for p in row[:h]:
            refs[p] += 1
    return refs


def _exact_attention(c, s, layer, table, lens, starts):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    parents = s["parents"].tolist() if s["parents"] is not None else None
    for b in range(c["slots"]):
        a, z = starts[b], starts[b + 1]
        n, end = z - a, lens[b] + z - a
        if not n:
            continue
        path = torch.ones(n, end, dtype=torch.bool)
        path[:, lens[b]:] = torch.ones(n, n).tril() > 0
        if parents is not None:
            for i in range(n):
                line = [i]
                while parents[a + line[-1]] >= 0:
                    line.append(parents[a + line[-1]])
                path[i, lens[b]:] = False
                path[i, [lens[b] + j for j in line]] = True
        path = path.cuda()
        ids = torch.tensor(table[b][:-(-end // c["page"])], device="cuda")
        for h in range(c["kv"]):
            k, v = (pool[layer, ids, h].reshape(-1, c["dim"])[:end].double() for pool in (s["k"], s["v"]))
            for q in range(h * c["groups"], (h + 1) * c["groups"]):
                x = (s["q"][a:z, q].double() @ k.T) / math.sqrt(c["dim"])
                out[a:z, q] = torch.softmax(x.masked_fill(~path, -math.inf), -1) @ v
    return out
