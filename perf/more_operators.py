"""The operators of serving sequences from a paged key/value cache and of checking a tree of drafted
tokens against the model: the append that rotates on the way, attention for steps, prompt chunks and
trees over the pages, and the acceptance that moves the kept tokens' rows into place.

`run` computes each in elementary torch operations, or, with `own` set, by the framework's kernels.
The cache: K and V [n_pages][n_head_kv][page][d] of 16-bit floats (f16 beside f32 rows, bf16 beside
bf16 rows) and an int32 table [n_batch][max_pages] of each sequence's pages, -1 where it has none yet.
A tree: int32 parents [n_batch][n], each below its own index, -1 for a root.
"""
import math

import torch

own = False

DEV = "cuda"
ROWS = {"f32": torch.float32, "bf16": torch.bfloat16}  # of a call's rows
HELD = {"f32": torch.float16, "bf16": torch.bfloat16}  # of the cache beside them
VOCAB = 151936


def listed():
    return [
        # one new token of 64 sequences: q and k rotated, k and v into pages of 16 tokens
        {"name": "append_step", "op": "append", "batch": 64, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "rot": 128,
         "type": "f32", "interleaved": False, "past": 2255, "page": 16, "tree": False, "ragged": True},
        # 24 drafted tokens of each of 16 sequences, at the positions of their depths
        {"name": "append_tree", "op": "append", "batch": 16, "n": 24, "heads": 14, "heads_kv": 2, "d": 64, "rot": 64,
         "type": "f32", "interleaved": False, "past": 1999, "page": 32, "tree": True, "ragged": True},
        # a prompt chunk of 64 sequences, interleaved pairs in the first half of the head
        {"name": "append_chunk", "op": "append", "batch": 64, "n": 256, "heads": 12, "heads_kv": 2, "d": 128, "rot": 64,
         "type": "bf16", "interleaved": True, "past": 1744, "page": 64, "tree": False, "ragged": False},
        # one user: a step after 2255 tokens
        {"name": "attn_step_one", "op": "attn", "batch": 1, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "type": "bf16",
         "past": 2255, "page": 16, "tree": False, "ragged": False, "padded": False},
        # the batch of 64 sequences at the middle of its decode
        {"name": "attn_step_64", "op": "attn", "batch": 64, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "type": "f32",
         "past": 2255, "page": 16, "tree": False, "ragged": False, "padded": False},
        # two very long contexts
        {"name": "attn_step_long", "op": "attn", "batch": 2, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "type": "bf16",
         "past": 131000, "page": 128, "tree": False, "ragged": False, "padded": False},
        # the last chunks of 2000-token prompts
        {"name": "attn_chunk_d128", "op": "attn", "batch": 32, "n": 256, "heads": 12, "heads_kv": 2, "d": 128,
         "type": "bf16", "past": 1744, "page": 64, "tree": False, "ragged": False, "padded": False},
        # a chunk of sequences of different lengths, padded on the left
        {"name": "attn_chunk_d64", "op": "attn", "batch": 16, "n": 250, "heads": 14, "heads_kv": 2, "d": 64,
         "type": "f32", "past": 1750, "page": 32, "tree": False, "ragged": True, "padded": True},
        # one user: 25 drafted tokens after 2255
        {"name": "attn_tree_one", "op": "attn", "batch": 1, "n": 25, "heads": 12, "heads_kv": 2, "d": 128, "type": "f32",
         "past": 2255, "page": 16, "tree": True, "ragged": False, "padded": False},
        # up to 61 drafted tokens of each of 32 sequences of different lengths
        {"name": "attn_tree_32", "op": "attn", "batch": 32, "n": 61, "heads": 14, "heads_kv": 2, "d": 64, "type": "bf16",
         "past": 4001, "page": 16, "tree": True, "ragged": True, "padded": True},
        # one user's drafted tokens after the model's answer: up to 7 of 25 stay, in the 28 layers' caches
        {"name": "keep_one", "op": "keep", "batch": 1, "n": 25, "heads_kv": 2, "d": 128, "type": "f32", "past": 205,
         "page": 16, "layers": 28, "kept": 7},
        # 64 sequences' drafted tokens: up to 9 of 61 stay, in 24 layers
        {"name": "keep_64", "op": "keep", "batch": 64, "n": 61, "heads_kv": 2, "d": 64, "type": "bf16", "past": 99,
         "page": 32, "layers": 24, "kept": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attn", "attn", "attn", "attn", "keep"])
    heads_kv = rng.choice([1, 2, 4, 8])
    heads, d = heads_kv * rng.choice([1, 2, 4, 6, 7, 8]), rng.choice([64, 128])
    kind, batch, page = rng.choice(["f32", "bf16"]), _log(rng, 1, 64), rng.choice([16, 32, 64, 128, 256])
    c = {"op": op, "batch": batch, "heads_kv": heads_kv, "d": d, "type": kind, "page": page}
    if op == "keep":
        c.update(heads_kv=min(heads_kv, 2), n=_log(rng, 1, 128), past=_log(rng, 1, 250), layers=rng.randint(1, 28))
        c["kept"] = rng.randint(1, min(c["n"], 12))
        return c
    if op == "append":
        shape = rng.choice(["step", "tree", "chunk"])
        c.update(heads=min(heads, 14), heads_kv=min(heads_kv, 2), past=_log(rng, 1, 4000), tree=shape == "tree",
                 rot=rng.choice([d, d // 2, d // 4, 24]), interleaved=rng.random() < 0.5, ragged=rng.random() < 0.5)
        c["heads"] = c["heads"] // c["heads_kv"] * c["heads_kv"]
        c["n"] = {"step": 1, "tree": _log(rng, 2, 128), "chunk": _log(rng, 2, 256)}[shape]
        return c
    shape = rng.choice(["step", "step", "few", "chunk", "tree", "tree"])
    n = {"step": 1, "few": rng.randint(2, 12), "chunk": _log(rng, 13, 256), "tree": _log(rng, 2, 128)}[shape]
    past = _log(rng, 1, 1744) if shape == "chunk" else _log(rng, 1, 131000)
    # no more keys and values than the longest listed step, no more products than the largest listed chunk
    batch = max(1, min(batch, 262000 // (past + n) * 2 // heads_kv))
    while batch > 1 and batch * heads * n * (past + n) * d > 32 * 12 * 256 * 2000 * 128:
        batch //= 2
    if batch * heads * n * (past + n) * d > 32 * 12 * 256 * 2000 * 128:
        n, shape = 1, "step"
    c.update(batch=batch, heads=heads, n=n, past=past, tree=shape == "tree", ragged=rng.random() < 0.4,
             padded=rng.random() < 0.4)
    return c


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _pages(c):
    """Pages a sequence's last token reaches."""
    return (c["past"] + c["n"] + c["page"] - 1) // c["page"]


def _table(g, c):
    """Each sequence's pages, handed out in no order from a pool with a few to spare, and room for
    more pages than it has."""
    B, mine = c["batch"], _pages(c)
    pool = B * mine + 5
    order = torch.randperm(pool, generator=g, device=DEV)[:B * mine].to(torch.int32)
    table = torch.full((B, mine + 3), -1, dtype=torch.int32, device=DEV)
    table[:, :mine] = order.view(B, mine)
    return table, pool


def _pool(g, c, pool, keys):
    """One side of the cache: keys with a few strong channels, values that differ along the pages."""
    H, page, d = c["heads_kv"], c["page"], c["d"]
    size = torch.exp(0.4 * (_normal(g, H, 1, d) if keys else _normal(g, pool, H, page, 1)))
    return (_normal(g, pool, H, page, d) * size).to(HELD[c["type"]])


def _tree(g, c):
    """A tree for each sequence, as a drafter grows one: a root, and later tokens below earlier ones."""
    B, n = c["batch"], c["n"]
    i = torch.arange(n, device=DEV)
    u = torch.rand(B, n, generator=g, device=DEV)
    return torch.minimum((u.sqrt() * i).long(), i - 1).to(torch.int32)  # (row 0: -1)


def _places(g, c):
    """Tokens before each sequence's new ones: a number, or for a ragged batch one for each."""
    if not c["ragged"]:
        return c["past"]
    t = torch.rand(c["batch"], generator=g, device=DEV)
    t = (t * (c["past"] + 1)).to(torch.int32).clamp_(max=c["past"])
    t[-1] = c["past"]
    return t


def _drafts(g, s, c):
    """Drafted tokens, their trees and the model's token after each: in every tree 1 to `kept` tokens,
    each below the one before, are what the model would have said."""
    B, n = c["batch"], c["n"]
    parent = _tree(g, c).long()
    tokens = torch.randint(0, VOCAB - 1, (B, n), generator=g, device=DEV)
    ids = torch.full((B, n), VOCAB - 1, device=DEV)  # a token that no draft holds
    kept = 1 + (torch.rand(B, generator=g, device=DEV) * c["kept"]).long().clamp_(max=c["kept"] - 1)
    # the chosen tokens of each tree: the root and kept - 1 others, in the order of their indices
    rank = torch.rand(B, n, generator=g, device=DEV)
    rank[:, 0] = -1
    chosen = rank.argsort(1).argsort(1) < kept[:, None]
    i = torch.arange(n, device=DEV)
    last = torch.where(chosen, i, -1).cummax(1).values           # the latest chosen one up to i
    before = torch.cat([torch.full((B, 1), -1, device=DEV), last[:, :-1]], 1)
    parent = torch.where(chosen, before, parent)
    b, j = torch.nonzero(chosen & (i > 0), as_tuple=True)
    ids[b, before[b, j]] = tokens[b, j]
    s["tree"], s["tokens"], s["ids"] = (t.to(torch.int32) for t in (parent, tokens, ids))


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV)
    g.manual_seed(seed)
    B, n, d, kind = c["batch"], c["n"], c["d"], ROWS[c["type"]]
    s = {"case": c}
    s["table"], pool = _table(g, c)
    if c["op"] == "keep":
        s["k"], s["v"] = ([_pool(g, c, pool, keys) for _ in range(c["layers"])] for keys in (True, False))
        _drafts(g, s, c)
        return s
    H, Hkv = c["heads"], c["heads_kv"]
    s["k"], s["v"] = _pool(g, c, pool, True), _pool(g, c, pool, False)
    s["past"] = _places(g, c)
    s["tree"] = _tree(g, c) if c["tree"] else None
    if c["op"] == "append":
        qkv = _normal(g, B, n, H + 2 * Hkv, d).to(kind)  # the packed projection
        s["q"], s["k_new"], s["v_new"] = qkv[:, :, :H], qkv[:, :, H:H + Hkv], qkv[:, :, H + Hkv:]
        s["q_out"] = torch.empty(B, n, H, d, dtype=kind, device=DEV)
        half = c["rot"] // 2
        speed = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        angle = torch.arange(c["past"] + n, dtype=torch.float64, device=DEV)[:, None] * speed
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s["count"] = s["first"] = None
    if c["padded"]:
        t = torch.rand(2, B, generator=g, device=DEV)
        s["count"] = n - (t[0] * 0.5 * n).to(torch.int32)
        s["first"] = (t[1] * 0.3 * s["past"]).to(torch.int32)
    s["q"] = (1.5 * _normal(g, B, n, H, d)).to(kind)
    s["out"] = (0.05 * _normal(g, B, n, H, d)).to(kind)  # rows behind a sequence's last token stay as they are
    return s


def run(state):
    return _run_own(state) if own else {"append": _append, "attn": _attn, "keep": _keep}[state["case"]["op"]](state)


def _run_own(s):
    from zwhisper_b200 import ops
    c = s["case"]
    if "cache" not in s:
        pools = zip(s["k"], s["v"]) if c["op"] == "keep" else [(s["k"], s["v"])]
        s["cache"] = [ops.PagedCache(k, v, s["table"]) for k, v in pools]
    cache = s["cache"][0]
    if c["op"] == "append":
        cache.append(s["k_new"], s["v_new"], s["past"], q=s["q"], q_out=s["q_out"], tree=s["tree"], max_past=c["past"],
                     rope=(s["cos"], s["sin"], c["interleaved"]))
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if c["op"] == "keep":
        path, kept, following = ops.tree_accept(s["tokens"], s["ids"], s["tree"])
        ops.paged_keep(s["cache"], path, kept, c["past"])
        return {"path": path, "kept": kept, "next": following, "k": s["k"], "v": s["v"]}
    return cache.attn(s["q"], s["past"], count=s["count"], first=s["first"], tree=s["tree"], max_past=c["past"],
                      out=s["out"])


def _above(parent):
    """above[b][i][j]: token j is i itself or one it descends from; and each token's depth."""
    n = parent.shape[1]
    i = torch.arange(n, device=DEV)
    step = ((parent[..., None] == i) | (i[:, None] == i)).float()  # to itself or one up
    for _ in range((n - 1).bit_length()):
        step = (step @ step > 0).float()
    return step > 0, (step.sum(-1) - 1).long()


def _row(past, batch, n):
    """Slots [batch][n] of the new tokens."""
    at = past if torch.is_tensor(past) else torch.full((batch,), past, device=DEV)
    return at.long()[:, None] + torch.arange(n, device=DEV)


def _append(s):
    c = s["case"]
    B, n, page = c["batch"], c["n"], c["page"]
    slot = _row(s["past"], B, n)
    at = slot[:, :1] + _above(s["tree"])[1] if c["tree"] else slot
    half = c["rot"] // 2
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    i = slice(0, c["rot"], 2) if c["interleaved"] else slice(0, half)
    j = slice(1, c["rot"], 2) if c["interleaved"] else slice(half, c["rot"])

    def turned(x):
        x = x.float()
        y = x.clone()
        y[..., i] = x[..., i] * cos - x[..., j] * sin
        y[..., j] = x[..., i] * sin + x[..., j] * cos
        return y

    s["q_out"].copy_(turned(s["q"]))
    where = s["table"].long().gather(1, slot // page), slice(None), slot % page
    s["k"][where] = turned(s["k_new"]).to(s["k"].dtype)
    s["v"][where] = s["v_new"].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _attn(s):
    c = s["case"]
    B, n, H, Hkv, d = c["batch"], c["n"], c["heads"], c["heads_kv"], c["d"]
    keys, group = c["past"] + n, H // Hkv
    pages = s["table"][:, :_pages(c)].long()
    k, v = (s[x][pages].transpose(1, 2).reshape(B, Hkv, -1, d)[:, :, :keys].float() for x in ("k", "v"))
    q = s["q"].float().view(B, n, Hkv, group, d).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * group, d)
    w = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).view(B, Hkv, n, group, keys)
    slot, j = _row(s["past"], B, n)[:, :, None], torch.arange(keys, device=DEV)
    if c["tree"]:
        mine = j - slot[:, :1]  # which of the call's tokens a key is
        own_token = (mine >= 0) & (mine < n)
        above = _above(s["tree"])[0].gather(2, mine.clamp(0, n - 1).expand(B, n, keys))
        seen = (mine < 0) | (own_token & above)
    else:
        seen = j <= slot
    if s["first"] is not None:
        seen = seen & (j >= s["first"][:, None, None])
    w.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(B, Hkv, n * group, keys) @ v).view(B, Hkv, n, group, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, H, d).to(s["out"].dtype)
    if s["count"] is not None:
        o = torch.where((torch.arange(n, device=DEV) < s["count"][:, None])[..., None, None], o, s["out"])
    s["out"].copy_(o)
    return s["out"]


def _keep(s):
    c = s["case"]
    B, n, page = c["batch"], c["n"], c["page"]
    i, b = torch.arange(n, device=DEV), torch.arange(B, device=DEV)
    parent, tokens, ids = s["tree"].long(), s["tokens"], s["ids"]
    at, alive = torch.zeros(B, dtype=torch.long, device=DEV), torch.ones(B, dtype=torch.bool, device=DEV)
    path = torch.full((B, n), -1, device=DEV)
    path[:, 0] = 0
    for step in range(1, n):
        fits = (parent == at[:, None]) & (tokens == ids[b, at][:, None]) & alive[:, None]
        alive = fits.any(1)
        at = torch.where(alive, torch.where(fits, i, n).amin(1), at)
        path[:, step] = torch.where(alive, at, -1)
    kept = (path >= 0).sum(1)
    dst = _row(c["past"], B, n)
    src = torch.where(path >= 0, dst[:, :1] + path, dst)  # a slot behind the kept ones: itself
    src_page, dst_page = (s["table"].long().gather(1, x // page) for x in (src, dst))
    for pool in s["k"] + s["v"]:
        pool[dst_page, :, dst % page] = pool[src_page, :, src % page]
    return {"path": path.to(torch.int32), "kept": kept.to(torch.int32), "next": ids[b, at].to(torch.int32), "k": s["k"],
            "v": s["v"]}


def _seen(c):
    """Pairs of a query and a key it sees, for the whole batch and one head, and the keys of one
    kv head that some query sees (a ragged batch: on average over its places)."""
    past = c["past"] / 2 if c["ragged"] else c["past"]
    count = 0.75 * c["n"] if c["padded"] and c["n"] > 1 else c["n"]
    first = 0.15 * past if c["padded"] else 0
    mine = 1 + math.log2(count) if c["tree"] else (count + 1) / 2  # of the call's own tokens
    return c["batch"] * count * (past - first + mine), c["batch"] * (past - first + count)


def work(case):
    c = case
    B, n, d, Hkv = c["batch"], c["n"], c["d"], c["heads_kv"]
    size = 4 if c["type"] == "f32" else 2
    if c["op"] == "keep":
        moved = B * (c["kept"] - 1) / 2 * c["layers"] * 2 * Hkv * d  # elements: a root stays where it is
        return {"bytes": 2 * moved * 2 + B * n * 16 + B * 8, "flops": B * n}
    if c["op"] == "append":
        q, kv = B * n * c["heads"] * d, B * n * Hkv * d
        tables = min(B * n, c["past"] + n) if c["ragged"] else n
        return {"bytes": 2 * q * size + 2 * kv * (size + 2) + tables * c["rot"] * 4 + (B * n * 4 if c["tree"] else 0),
                "flops": B * n * (c["heads"] + Hkv) * c["rot"] * 3}
    pairs, keys = _seen(c)
    return {"bytes": 2 * keys * Hkv * d * 2 + 2 * B * n * c["heads"] * d * size, "flops": 4 * pairs * c["heads"] * d}


def _lines(parent):
    """For each token of one tree, the indices from it up to its root."""
    up = parent.tolist()
    lines = []
    for i in range(len(up)):
        lines.append([i] + (lines[up[i]] if up[i] >= 0 else []))
    return lines


def exact(case, seed):
    """From the definitions, in 64 bits, one sequence after another."""
    c, s = case, prepare(case, seed)
    B, n, d, page = c["batch"], c["n"], c["d"], c["page"]
    table = s["table"].tolist()
    if c["op"] == "keep":
        k, v = ([p.double() for p in s[x]] for x in ("k", "v"))
        paths, follow = [], []
        for b in range(B):
            up, tok, ans = (s[x][b].tolist() for x in ("tree", "tokens", "ids"))
            path = [0]
            while True:
                below = [i for i in range(n) if up[i] == path[-1] and tok[i] == ans[path[-1]]]
                if not below:
                    break
                path.append(below[0])
            src = torch.tensor([c["past"] + i for i in path], device=DEV)
            dst = torch.arange(c["past"], c["past"] + len(path), device=DEV)
            mine = s["table"][b].long()
            for p in k + v:
                p[mine[dst // page], :, dst % page] = p[mine[src // page], :, src % page].clone()
            paths.append(path)
            follow.append(ans[path[-1]])
        return {"path": torch.tensor([p + [-1] * (n - len(p)) for p in paths], dtype=torch.int32),
                "kept": torch.tensor([len(p) for p in paths], dtype=torch.int32),
                "next": torch.tensor(follow, dtype=torch.int32), "k": k, "v": v}
    places = [int(s["past"][b]) if c["ragged"] else c["past"] for b in range(B)]
    lines = [_lines(s["tree"][b]) for b in range(B)] if c["tree"] else None
    if c["op"] == "append":
        k, v, q, half = s["k"].double(), s["v"].double(), s["q"].double(), c["rot"] // 2

        def turn(x, at):  # x [n][heads][d]
            pairs = x[..., :2 * half].reshape(*x.shape[:-1], *((half, 2) if c["interleaved"] else (2, half)))
            pairs = pairs if c["interleaved"] else pairs.transpose(-1, -2)
            z = torch.view_as_complex(pairs.contiguous())
            z = torch.view_as_real(z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None])
            z = z if c["interleaved"] else z.transpose(-1, -2)
            return torch.cat([z.reshape(*x.shape[:-1], 2 * half), x[..., 2 * half:]], -1)

        for b in range(B):
            depth = [len(line) - 1 for line in lines[b]] if c["tree"] else range(n)
            at = torch.tensor([places[b] + x for x in depth], device=DEV)
            q[b] = turn(q[b], at)
            k_new = turn(s["k_new"][b].double(), at)
            slot = torch.arange(places[b], places[b] + n, device=DEV)
            to = s["table"][b].long()[slot // page]
            k[to, :, slot % page] = k_new
            v[to, :, slot % page] = s["v_new"][b].double()
        return {"q": q, "k": k, "v": v}
    out, group = s["out"].double(), c["heads"] // c["heads_kv"]
    for b in range(B):
        past = places[b]
        count, first = (int(s["count"][b]), int(s["first"][b])) if c["padded"] else (n, 0)
        pages = table[b][:(past + count + page - 1) // page]
        seen = torch.zeros(count, past + count, dtype=torch.bool, device=DEV)
        if c["tree"]:
            seen[:, first:past] = True
            rows = [i for i in range(count) for _ in lines[b][i]]
            cols = [past + j for i in range(count) for j in lines[b][i]]
            seen[torch.tensor(rows, device=DEV), torch.tensor(cols, device=DEV)] = True
        else:
            for i in range(count):
                seen[i, first:past + i + 1] = True
        for h in range(c["heads_kv"]):
            k, v = (torch.cat([s[x][p, h] for p in pages]).double()[:past + count] for x in ("k", "v"))
            q = s["q"][b, :count, h * group:(h + 1) * group].double()
            w = torch.einsum("ngd,kd->ngk", q, k) / math.sqrt(d)
            w = w.masked_fill(~seen[:, None], -math.inf)
            out[b, :count, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", torch.softmax(w, -1), v)
    return out
