"""The operators of a decode step over a key/value cache held in 8 bits: rotary positions, the
append that quantises, the attention that reads the cache, and the rules on the logits.

`run` computes each in elementary torch operations, or, with `own` set, by the framework's
kernels. The cache: int8 K [n_batch][n_head_kv][blocks][32][d] and V [n_batch][n_head_kv][blocks]
[d][32] with one f32 scale for each block of 32 tokens and head; the last block's rows also in f32
(k_open, v_open [n_batch][n_head_kv][32][d], of block open_block [n_batch][n_head_kv]), so that its
int8 values always come from the original rows.
"""
import math

import torch

own = False

BLOCK = 32
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of each of 16 sequences, 14 + 2 heads of 64: q and k out of the packed projection
        {"name": "rope_step", "op": "rope", "batch": 16, "n": 1, "heads": 14, "heads_kv": 2, "d": 64, "rot": 64,
         "type": "f32", "interleaved": False, "past": 2255, "ragged": False},
        # a prompt chunk of 64 sequences, interleaved pairs in the first half of the head, each sequence at its own place
        {"name": "rope_chunk", "op": "rope", "batch": 64, "n": 256, "heads": 12, "heads_kv": 2, "d": 128, "rot": 64,
         "type": "bf16", "interleaved": True, "past": 1744, "ragged": True},
        # one new token of 64 sequences in the middle of a block
        {"name": "append_step", "op": "append", "batch": 64, "n": 1, "heads_kv": 2, "d": 128, "type": "f32", "past": 2255},
        # a prompt chunk of 64 sequences that starts and ends inside a block
        {"name": "append_chunk", "op": "append", "batch": 64, "n": 256, "heads_kv": 2, "d": 128, "type": "f32", "past": 1741},
        # one user: a step after 2255 tokens
        {"name": "attn_step_one", "op": "attn", "batch": 1, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "type": "f32",
         "past": 2255, "ragged": False, "padded": False},
        # the batch of 64 sequences at the middle of its decode
        {"name": "attn_step_64", "op": "attn", "batch": 64, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "type": "f32",
         "past": 2255, "ragged": False, "padded": False},
        # sequences of different lengths, padded on the left
        {"name": "attn_step_ragged", "op": "attn", "batch": 16, "n": 1, "heads": 14, "heads_kv": 2, "d": 64,
         "type": "bf16", "past": 4001, "ragged": True, "padded": True},
        # two very long contexts
        {"name": "attn_step_long", "op": "attn", "batch": 2, "n": 1, "heads": 12, "heads_kv": 2, "d": 128, "type": "bf16",
         "past": 131000, "ragged": False, "padded": False},
        # the last chunks of 2000-token prompts
        {"name": "attn_chunk_d128", "op": "attn", "batch": 32, "n": 256, "heads": 12, "heads_kv": 2, "d": 128,
         "type": "f32", "past": 1744, "ragged": False, "padded": False},
        # a chunk whose sequences end at different tokens
        {"name": "attn_chunk_d64", "op": "attn", "batch": 16, "n": 250, "heads": 14, "heads_kv": 2, "d": 64,
         "type": "bf16", "past": 1750, "ragged": True, "padded": True},
        # one row of a 151936-token vocabulary under a grammar, after a short answer
        {"name": "logits_one", "op": "logits", "batch": 1, "vocab": 151936, "recent": 300, "window": 256, "bias": 32,
         "mask": True},
        # a batch of 64 rows with long histories
        {"name": "logits_64", "op": "logits", "batch": 64, "vocab": 151936, "recent": 2000, "window": 1024, "bias": 300,
         "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "attn", "logits"])
    heads_kv = rng.choice([1, 2, 4, 8])
    heads, d = heads_kv * rng.choice([1, 2, 4, 6, 7, 8]), rng.choice([64, 128])
    kind, batch = rng.choice(["f32", "bf16"]), _log(rng, 1, 64)
    if op == "logits":
        recent = _log(rng, 1, 4000)
        return {"op": op, "batch": batch, "vocab": _log(rng, 1000, 151936), "recent": recent,
                "window": _log(rng, 1, recent), "bias": rng.choice([0, _log(rng, 1, 300)]), "mask": rng.random() < 0.6}
    if op == "rope":
        n = 1 if rng.random() < 0.5 else _log(rng, 2, 256)
        return {"op": op, "batch": batch, "n": n, "heads": min(heads, 14), "heads_kv": min(heads_kv, 2), "d": d,
                "rot": rng.choice([d, d // 2, d // 4, 24]), "type": kind, "interleaved": rng.random() < 0.5,
                "past": _log(rng, 1, 8000), "ragged": rng.random() < 0.5}
    if op == "append":
        n = 1 if rng.random() < 0.5 else _log(rng, 2, 256)
        return {"op": op, "batch": batch, "n": n, "heads_kv": min(heads_kv, 2), "d": d, "type": kind,
                "past": _log(rng, 1, 4000)}
    shape = rng.choice(["step", "step", "few", "chunk"])
    n = {"step": 1, "few": rng.randint(2, 12), "chunk": _log(rng, 13, 256)}[shape]
    past = _log(rng, 1, 1744) if shape == "chunk" else _log(rng, 1, 131000)
    # no more keys and values than the longest listed step, no more products than the largest listed chunk
    batch = max(1, min(batch, 262000 // (past + n) * 2 // heads_kv))
    while batch > 1 and batch * heads * n * (past + n) * d > 32 * 12 * 256 * 2000 * 128:
        batch //= 2
    if batch * heads * n * (past + n) * d > 32 * 12 * 256 * 2000 * 128:
        n = 1
    return {"op": op, "batch": batch, "n": n, "heads": heads, "heads_kv": heads_kv, "d": d, "type": kind, "past": past,
            "ragged": rng.random() < 0.4, "padded": rng.random() < 0.4}


def _ctx(c):
    """Tokens a cache or a table has room for: a little more than the case fills."""
    return (c["past"] + c["n"] + 95) // BLOCK * BLOCK


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _quantised(x):
    """int8 values and f32 scales of x [..., 32, d], one scale for the last two dimensions; in 64
    bits, since a value next to the border between two integers goes by its last bit."""
    top = x.abs().amax(dim=(-1, -2))
    over = torch.where(top > 0, top, 1.0).double()[..., None, None]
    return torch.round(127.0 * x.double() / over).to(torch.int8), top / 127.0


def _cache(g, c):
    """A cache of c["past"] tokens, one head after another (keys with a few strong channels, values
    whose size changes along the context, as projections give them)."""
    B, H, d, past, nb = c["batch"], c["heads_kv"], c["d"], c["past"], _ctx(c) // BLOCK
    s = {"k": torch.empty(B, H, nb, BLOCK, d, dtype=torch.int8, device=DEV),
         "v": torch.empty(B, H, nb, d, BLOCK, dtype=torch.int8, device=DEV),
         "k_scale": torch.empty(B, H, nb, device=DEV), "v_scale": torch.empty(B, H, nb, device=DEV)}
    opened = []
    for name in ("k", "v"):
        size = torch.exp(0.4 * _normal(g, H, 1, d)) if name == "k" else torch.exp(0.4 * _normal(g, H, nb * BLOCK, 1))
        tail = torch.zeros(B, H, BLOCK, d, device=DEV)
        for b in range(B):
            x = _normal(g, H, nb * BLOCK, d) * size
            x[:, past:] = 0
            q, t = _quantised(x.view(H, nb, BLOCK, d))
            s[name][b] = q if name == "k" else q.transpose(-1, -2)
            s[name + "_scale"][b] = t
            at = past // BLOCK * BLOCK
            tail[b] = x[:, at:at + BLOCK]
        opened.append(tail)
    s["k_open"], s["v_open"] = opened
    s["open_block"] = torch.full((B, H), past // BLOCK, dtype=torch.int32, device=DEV)
    return s


def _places(g, c):
    """Tokens before each sequence's new ones: a number, or for a ragged batch one for each."""
    if not c["ragged"]:
        return c["past"]
    t = torch.rand(c["batch"], generator=g, device=DEV)
    t = (t * (c["past"] + 1)).to(torch.int32).clamp_(max=c["past"])
    t[-1] = c["past"]
    return t


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "logits":
        B, V = c["batch"], c["vocab"]
        s["logits"] = 3 * _normal(g, B, V)
        # words of a text: few are frequent, most are rare
        word = torch.rand(B, c["recent"], generator=g, device=DEV) ** 4 * V
        s["recent"] = word.to(torch.int32).clamp_(max=V - 1)
        s["bias_ids"] = torch.randint(0, V, (c["bias"],), generator=g, device=DEV, dtype=torch.int32)
        s["bias"] = 2 * _normal(g, c["bias"])
        # a grammar lets through a few tokens, or most of them
        share = torch.rand(B, 1, generator=g, device=DEV)
        bits = torch.rand(B, (V + 31) // 32, 32, generator=g, device=DEV) < share[..., None]
        word = (bits.long() << torch.arange(32, device=DEV)).sum(-1)
        s["allow"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32) if c["mask"] else None
        return s
    B, n, d, kind = c["batch"], c["n"], c["d"], TYPES[c["type"]]
    if c["op"] == "rope":
        H, Hkv = c["heads"], c["heads_kv"]
        s["past"] = _places(g, c)
        qkv = _normal(g, B, n, H + 2 * Hkv, d).to(kind)  # the packed projection of a chunk
        s["q"], s["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
        half = c["rot"] // 2
        speed = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        speed = torch.where(speed < 1e-3, speed / 4, speed)  # slow turns slowed down further: a longer context
        angle = torch.arange(_ctx(c), dtype=torch.float64, device=DEV)[:, None] * speed
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s.update(_cache(g, c))
    if c["op"] == "append":
        s["k_new"], s["v_new"] = ((2 * _normal(g, B, n, c["heads_kv"], d)).to(kind) for _ in range(2))
        return s
    s["past"] = _places(g, c)
    s["count"] = s["first"] = None
    if c["padded"]:
        t = torch.rand(2, B, generator=g, device=DEV)
        s["count"] = n - (t[0] * 0.5 * n).to(torch.int32)
        s["first"] = (t[1] * 0.3 * s["past"]).to(torch.int32)
    s["q"] = (1.5 * _normal(g, B, n, c["heads"], d)).to(kind)
    s["out"] = (0.05 * _normal(g, B, n, c["heads"], d)).to(kind)  # rows behind a sequence's last token stay as they are
    return s


def run(state):
    return _run_own(state) if own else {"rope": _rope, "append": _append, "attn": _attn, "logits": _logits}[state["case"]["op"]](state)


def _run_own(s):
    from zwhisper_b200 import ops
    c = s["case"]
    if c["op"] == "rope":
        q, k = ops.rope(s["q"], s["cos"], s["sin"], s["past"], k=s["k"], interleaved=c["interleaved"], inplace=False)
        return {"q": q, "k": k}
    if c["op"] == "logits":
        ids = ops.llm_logits(s["logits"], recent=s["recent"], window=c["window"], repeat=1.1, presence=0.3, frequency=0.2,
                             bias_ids=s["bias_ids"], bias=s["bias"], allow=s["allow"])
        return {"logits": s["logits"], "ids": ids}
    if "cache" not in s:
        s["cache"] = ops.Kv8Cache(s["k"], s["k_scale"], s["v"], s["v_scale"], s["k_open"], s["v_open"], s["open_block"])
    cache = s["cache"]
    if c["op"] == "append":
        cache.append(s["k_new"], s["v_new"], c["past"])
        at = c["past"] // BLOCK * BLOCK
        k, v = cache.read(c["past"] + c["n"] - at, at)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "k_open": s["k_open"],
                "v_open": s["v_open"]}
    return cache.attn(s["q"], s["past"], count=s["count"], first=s["first"], max_past=c["past"], out=s["out"])


def _row(past, batch, n):
    """Positions [batch][n] of the new tokens."""
    at = past if torch.is_tensor(past) else torch.full((batch,), past, device=DEV)
    return at.long()[:, None] + torch.arange(n, device=DEV)


def _rope(s):
    c, out = s["case"], {}
    half, at = c["rot"] // 2, _row(s["past"], c["batch"], c["n"])
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    for name in ("q", "k"):
        x = s[name].float()
        y = x.clone()
        i = slice(0, c["rot"], 2) if c["interleaved"] else slice(0, half)
        j = slice(1, c["rot"], 2) if c["interleaved"] else slice(half, c["rot"])
        y[..., i] = x[..., i] * cos - x[..., j] * sin
        y[..., j] = x[..., i] * sin + x[..., j] * cos
        out[name] = y.to(s[name].dtype)
    return out


def _append(s):
    c, out = s["case"], {}
    B, H, d, past, n = c["batch"], c["heads_kv"], c["d"], c["past"], c["n"]
    b0, b1, held = past // BLOCK, (past + n - 1) // BLOCK, past % BLOCK
    for name in ("k", "v"):
        ints, scale, tail, new = s[name], s[name + "_scale"], s[name + "_open"], s[name + "_new"]
        rows = torch.zeros(B, H, (b1 - b0 + 1) * BLOCK, d, device=DEV)
        if held:  # the open block's rows, or what the cache stands for where it went back into a full one
            old = (ints[:, :, b0] if name == "k" else ints[:, :, b0].transpose(-1, -2)).float() * scale[:, :, b0, None, None]
            mine = (s["open_block"] == b0)[..., None, None]
            rows[:, :, :held] = torch.where(mine, tail, old)[:, :, :held]
        rows[:, :, held:held + n] = new.float().transpose(1, 2)
        blocks = rows.view(B, H, -1, BLOCK, d)
        q, t = _quantised(blocks)
        ints[:, :, b0:b1 + 1] = q if name == "k" else q.transpose(-1, -2)
        scale[:, :, b0:b1 + 1] = t
        tail.copy_(blocks[:, :, -1])
        values = q.float() * t[..., None, None]
        out[name] = values.view(B, H, -1, d)[:, :, :held + n].transpose(1, 2).contiguous()
        out[name + "_scale"], out[name + "_open"] = scale, tail
    s["open_block"].fill_(b1)
    return out


def _attn(s):
    c = s["case"]
    B, n, H, Hkv, d = c["batch"], c["n"], c["heads"], c["heads_kv"], c["d"]
    keys, group = c["past"] + n, H // Hkv
    nb = (keys + BLOCK - 1) // BLOCK
    k = s["k"][:, :, :nb].float() * s["k_scale"][:, :, :nb, None, None]
    v = (s["v"][:, :, :nb].float() * s["v_scale"][:, :, :nb, None, None]).transpose(-1, -2)
    k, v = k.reshape(B, Hkv, nb * BLOCK, d)[:, :, :keys], v.reshape(B, Hkv, nb * BLOCK, d)[:, :, :keys]
    q = s["q"].float().view(B, n, Hkv, group, d).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * group, d)
    w = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).view(B, Hkv, n, group, keys)
    at, j = _row(s["past"], B, n)[:, :, None], torch.arange(keys, device=DEV)
    seen = j <= at
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


def _logits(s):
    c, x = s["case"], s["logits"]
    B, V = c["batch"], c["vocab"]
    window = s["recent"][:, max(0, c["recent"] - c["window"]):].long()
    times = torch.zeros(B, V, device=DEV).scatter_add_(1, window, torch.ones_like(window, dtype=torch.float32))
    y = torch.where(x > 0, x / 1.1, x * 1.1) - (times * 0.2 + 0.3)
    y = torch.where(times > 0, y, x)
    if c["bias"]:
        y = y + torch.zeros(V, device=DEV).index_add_(0, s["bias_ids"].long(), s["bias"])
    if s["allow"] is not None:
        bits = (s["allow"][..., None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        y = torch.where(bits.view(B, -1)[:, :V] != 0, y, -math.inf)
    x.copy_(y)
    top, ids = x.max(dim=1)
    ids = torch.where(top > -math.inf, (x == top[:, None]).int().argmax(1), -1)
    return {"logits": x, "ids": ids.to(torch.int32)}


def _seen(c):
    """Pairs of a query and a key it sees, for the whole batch and one head, and the keys of one
    kv head that some query sees (a ragged batch: on average over its places)."""
    past = c["past"] / 2 if c["ragged"] else c["past"]
    count = 0.75 * c["n"] if c["padded"] and c["n"] > 1 else c["n"]
    first = 0.15 * past if c["padded"] else 0
    return c["batch"] * count * (past - first + (count + 1) / 2), c["batch"] * (past - first + count)


def work(case):
    c = case
    if c["op"] == "logits":
        rows = c["batch"] * c["vocab"]
        lists = c["batch"] * min(c["recent"], c["window"]) * 4 + c["bias"] * 8
        return {"bytes": 8 * rows + (rows / 8 if c["mask"] else 0) + lists, "flops": rows}
    size = 4 if c["type"] == "f32" else 2
    B, n, d = c["batch"], c["n"], c["d"]
    if c["op"] == "rope":
        values = B * n * (c["heads"] + c["heads_kv"])
        tables = min(B * n, _ctx(c)) if c["ragged"] else n
        return {"bytes": 2 * values * d * size + tables * c["rot"] * 4, "flops": values * c["rot"] * 3}
    if c["op"] == "append":
        new, held = B * n * c["heads_kv"] * d, c["past"] % BLOCK
        rows = B * c["heads_kv"] * d * (held + n)
        # K and V: new rows in, the open block's rows in and out, ints out; the ints in and their values out again
        return {"bytes": 2 * (new * size + B * c["heads_kv"] * d * (held + (held + n) % BLOCK) * 4 + rows * (1 + 1 + 4)),
                "flops": 2 * rows * 4}
    pairs, keys = _seen(c)
    return {"bytes": 2 * keys * c["heads_kv"] * (d + 4 / BLOCK) + 2 * B * n * c["heads"] * d * size,
            "flops": 4 * pairs * c["heads"] * d}


def exact(case, seed):
    """From the definitions, in 64 bits, one sequence and head after another."""
    c, s = case, prepare(case, seed)
    if c["op"] == "logits":
        rows, ids = [], []
        for b in range(c["batch"]):
            x = s["logits"][b].double()
            for_row = s["recent"][b, -min(c["window"], c["recent"]):].long()
            word, times = torch.unique(for_row, return_counts=True)
            hit = x[word]
            # the rules' numbers as the kernels get them: f32
            r, p, f = (float(torch.tensor(v, dtype=torch.float32)) for v in (1.1, 0.3, 0.2))
            x[word] = torch.where(hit > 0, hit / r, hit * r) - f * times - p
            x.index_put_((s["bias_ids"].long(),), s["bias"].double(), accumulate=True)
            if s["allow"] is not None:
                t = torch.arange(c["vocab"], device=DEV)
                x[(s["allow"][b].long()[t // 32] >> (t % 32)) % 2 == 0] = -math.inf
            rows.append(x)
            ids.append(int(x.argmax()) if bool((x > -math.inf).any()) else -1)
        return {"logits": torch.stack(rows), "ids": torch.tensor(ids, dtype=torch.int32)}
    B, n, d = c["batch"], c["n"], c["d"]
    if c["op"] == "rope":
        out, half = {}, c["rot"] // 2
        at = [int(s["past"][b]) if c["ragged"] else c["past"] for b in range(B)]
        turn = torch.stack([torch.complex(s["cos"][a:a + n].double(), s["sin"][a:a + n].double()) for a in at])
        for name in ("q", "k"):
            x = s[name].double()
            pairs = x[..., :c["rot"]].reshape(*x.shape[:-1], *((half, 2) if c["interleaved"] else (2, half)))
            pairs = pairs if c["interleaved"] else pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, :, None])
            z = z if c["interleaved"] else z.transpose(-1, -2)
            out[name] = torch.cat([z.reshape(*x.shape[:-1], c["rot"]), x[..., c["rot"]:]], -1)
        return out
    if c["op"] == "append":
        out = {}
        begin, end = c["past"] // BLOCK * BLOCK, c["past"] + n
        for name in ("k", "v"):
            held = s[name + "_open"][:, :, :c["past"] - begin].double()
            x = torch.cat([held, s[name + "_new"].double().permute(0, 2, 1, 3)], 2)
            scale, values = s[name + "_scale"].double(), torch.empty_like(x)
            for i in range(0, end - begin, BLOCK):
                part = x[:, :, i:i + BLOCK]
                top = part.abs().flatten(2).max(-1).values[..., None, None]
                values[:, :, i:i + BLOCK] = torch.round(part * 127 / top) * top / 127
                scale[:, :, (begin + i) // BLOCK] = top[..., 0, 0] / 127
            last = (end - 1) // BLOCK * BLOCK - begin
            tail = torch.zeros(B, c["heads_kv"], BLOCK, d, dtype=torch.float64, device=DEV)
            tail[:, :, :end - begin - last] = x[:, :, last:]
            out[name], out[name + "_scale"], out[name + "_open"] = values.transpose(1, 2), scale, tail
        return out
    out, group = s["out"].double(), c["heads"] // c["heads_kv"]
    for b in range(B):
        past = int(s["past"][b]) if c["ragged"] else c["past"]
        count, first = (int(s["count"][b]), int(s["first"][b])) if c["padded"] else (n, 0)
        for h in range(c["heads_kv"]):
            k = (s["k"][b, h].double() * s["k_scale"][b, h].double()[:, None, None]).reshape(-1, d)[first:past + count]
            v = s["v"][b, h].double() * s["v_scale"][b, h].double()[:, None, None]
            v = v.transpose(-1, -2).reshape(-1, d)[first:past + count]
            q = s["q"][b, :count, h * group:(h + 1) * group].double()
            w = torch.einsum("ngd,kd->ngk", q, k) / math.sqrt(d)
            for i in range(count):
                w[i, :, past + i + 1 - first:] = -math.inf
            out[b, :count, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", torch.softmax(w, -1), v)
    return out
