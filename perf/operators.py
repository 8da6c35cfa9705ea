"""Measured cases of the decode-step operators around the quantized projections:

  plan     block table, slot map, positions and lengths of a step, built on the GPU from the sequences' lengths
  append   rotary positions on a step's queries and keys, keys and values appended to the paged 8-bit cache
  attn     attention of a step's queries over the paged 8-bit cache
  sample   tokens drawn from logits with temperature, top-k, top-p and min-p from given random numbers

`own` chooses between the plain form (elementary torch operations) and the framework's kernels; both take the state
that prepare() makes.  The cache holds int8 codes with one float scale per block of tokens and head, for keys and for
values; the scales written by an append are powers of two."""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"


def listed():
    return [
        # one token for each of a few running sequences: what every small decode step does first
        {"name": "plan, 8 decoding", "op": "plan", "seqs": 8, "new": 1, "prompts": 0, "done": 0, "ctx": 2000, "block": 16, "ragged": 1},
        # a full server step: decoding sequences, some prompts of up to 1536 tokens, some finished ones giving blocks back
        {"name": "plan, 1024 mixed", "op": "plan", "seqs": 1024, "new": 1, "prompts": 24, "done": 9, "ctx": 6000, "block": 16, "ragged": 2},
        # a decode step of eight sequences, heads of the 70B-shaped stack
        {"name": "append, 8 decoding", "op": "append", "seqs": 8, "new": 1, "qh": 64, "kvh": 8, "dim": 128, "rot": 128, "pairs": False, "block": 16, "ctx": 1500, "f32": False, "ragged": 3},
        # a prompt of 8192 tokens, heads of the 8B-shaped stack
        {"name": "append, prompt 8192", "op": "append", "seqs": 1, "new": 8192, "qh": 32, "kvh": 8, "dim": 128, "rot": 128, "pairs": False, "block": 64, "ctx": 0, "f32": False, "ragged": 4},
        # ragged chunks of float32 activations, part of an interleaved head rotated
        {"name": "append, ragged f32", "op": "append", "seqs": 13, "new": 61, "qh": 21, "kvh": 3, "dim": 64, "rot": 32, "pairs": True, "block": 32, "ctx": 700, "f32": True, "ragged": 5},
        # one sequence, one token: latency of a single user
        {"name": "attn, 1 x 1", "op": "attn", "seqs": 1, "new": 1, "qh": 64, "kvh": 8, "dim": 128, "block": 16, "ctx": 8191, "window": 0, "f32": False, "ragged": 6},
        # a batch of decoding sequences of ragged lengths: the bandwidth case
        {"name": "attn, 64 decoding", "op": "attn", "seqs": 64, "new": 1, "qh": 64, "kvh": 8, "dim": 128, "block": 64, "ctx": 12000, "window": 0, "f32": False, "ragged": 7},
        # a chunk of a long prompt: the arithmetic case
        {"name": "attn, prompt 4096", "op": "attn", "seqs": 1, "new": 4096, "qh": 32, "kvh": 8, "dim": 128, "block": 64, "ctx": 4096, "window": 0, "f32": False, "ragged": 8},
        # short drafts to be verified, odd lengths, a sliding window, float32 activations
        {"name": "attn, drafts f32", "op": "attn", "seqs": 19, "new": 5, "qh": 21, "kvh": 3, "dim": 64, "block": 32, "ctx": 3001, "window": 1000, "f32": True, "ragged": 9},
        # one row of a small vocabulary
        {"name": "sample, 1 x 32000", "op": "sample", "rows": 1, "vocab": 32000, "f32": False, "cut": "kp", "ragged": 10},
        # a decode batch over a large vocabulary, every filter in use
        {"name": "sample, 64 x 131072", "op": "sample", "rows": 64, "vocab": 131072, "f32": False, "cut": "kpm", "ragged": 11},
        # many rows, an odd vocabulary, float32 logits, no top-k
        {"name": "sample, 200 x 50257", "op": "sample", "rows": 200, "vocab": 50257, "f32": True, "cut": "pm", "ragged": 12},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attn", "attn", "attn", "sample", "sample"])
    ragged = rng.randrange(1 << 20)
    if op == "plan":
        seqs = _log(rng, 1, 1024)
        return {"op": op, "seqs": seqs, "new": rng.choice([1, 1, 2, 5]), "prompts": rng.randint(0, min(16, seqs // 8)), "done": rng.randint(0, seqs // 16), "ctx": _log(rng, 20, 6000),
                "block": rng.choice([16, 32, 64, 128]), "ragged": ragged}
    if op == "sample":
        vocab = _log(rng, 1000, 131072)
        return {"op": op, "rows": _log(rng, 1, min(256, 64 * 131072 // vocab)), "vocab": vocab, "f32": rng.random() < 0.4, "cut": rng.choice(["", "k", "p", "m", "kp", "pm", "kpm"]), "ragged": ragged}
    kvh = rng.choice([1, 2, 3, 4, 8])
    qh, dim, block, f32 = kvh * rng.choice([1, 2, 4, 5, 7, 8]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128]), rng.random() < 0.25
    if op == "append":
        seqs = _log(rng, 1, 64)
        return {"op": op, "seqs": seqs, "new": _log(rng, 1, 4096 // seqs), "qh": qh, "kvh": kvh, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "pairs": rng.random() < 0.4,
                "block": block, "ctx": _log(rng, 1, 4000), "f32": f32, "ragged": ragged}
    if rng.random() < 0.6:
        seqs, new, ctx = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7]), _log(rng, 30, 12000)
    else:
        seqs, new = rng.randint(1, 4), _log(rng, 8, 1024)
        ctx = new + _log(rng, 1, 4000)
    return {"op": op, "seqs": seqs, "new": new, "qh": qh, "kvh": kvh, "dim": dim, "block": block, "ctx": ctx, "window": rng.choice([0, 0, 0, 128, 1000]), "f32": f32, "ragged": ragged}


def _lengths(case):
    """(tokens cached before the step, tokens of the step) of each sequence, from the case alone."""
    rng = random.Random(case["ragged"])
    n, ctx, new = case["seqs"], case["ctx"], case["new"]
    if case["op"] == "plan":
        old = [rng.randint(ctx // 4, ctx) for _ in range(n)]
        add = [new] * n
        for i in rng.sample(range(n), case["prompts"] + case["done"]):
            add[i], old[i] = (rng.randint(200, 1536), rng.choice([0, 0, old[i]]))
        for i in rng.sample(range(n), case["done"]):
            add[i] = -1
        return old, add
    if case["op"] == "append":
        return [rng.randint(0, ctx) for _ in range(n)], [new if new == 1 or n == 1 else rng.randint(0, 2 * new) for _ in range(n)]
    # attention: `ctx` and `new` are the largest of their kind; now and then a sequence brings no token
    old, add = [], []
    for i in range(n):
        t = new if i == 0 or new == 1 else rng.randint(0, new)
        old.append(ctx if i == 0 else rng.randint(ctx // 4, ctx))
        add.append(t)
    return old, add


def _up(a, b):
    return -(-a // b)


def _pool(gen, old, add, block, spare=0):
    """Blocks for every sequence's tokens, in random order: (block table, blocks in the pool)."""
    need = [_up(o + max(a, 0), block) for o, a in zip(old, add)]
    width, total = max(1, max(need)), sum(need) + spare
    order = torch.randperm(max(total, 1), generator=gen, device=DEV).to(torch.int32)
    first = torch.tensor(np.concatenate([[0], np.cumsum(need)[:-1]]), device=DEV)
    col = torch.arange(width, device=DEV)
    index = (first[:, None] + col).clamp(max=max(total, 1) - 1)
    return torch.where(col < torch.tensor(need, device=DEV)[:, None], order[index], torch.full_like(order[index], -1)), max(total, 1)


def _cache(gen, blocks, kvh, block, dim):
    shape = (blocks, kvh, block, dim)

    def codes():
        x = torch.empty(shape, dtype=torch.int8, device=DEV)
        for i in range(0, blocks, 4096):
            x[i:i + 4096] = (torch.randn(x[i:i + 4096].shape, generator=gen, device=DEV) * 30).round().clamp(-127, 127).to(torch.int8)
        return x

    def scales():
        return torch.exp2(torch.randint(-6, -4, (blocks, kvh), generator=gen, device=DEV).float())

    return {"k": codes(), "v": codes(), "k_scale": scales(), "v_scale": scales()}


def _frequencies(dim, base=500000.0):
    """A long-context model's frequencies: the slow ones stretched eightfold, with a ramp between."""
    f = base ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    turns = 8192 * f / (2 * math.pi)
    keep = np.clip((turns - 1) / (4 - 1), 0, 1)
    return f * keep + f / 8 * (1 - keep)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device=DEV) * 2
        x += 5 * (torch.rand(rows, vocab, generator=gen, device=DEV) < 0.002)
        x[torch.rand(rows, vocab, generator=gen, device=DEV) < 0.01] = -math.inf  # tokens that a grammar forbids
        pick = lambda v: torch.tensor(v, device=DEV)[torch.randint(0, len(v), (rows,), generator=gen, device=DEV)]  # noqa: E731
        s = {"logits": x if case["f32"] else x.half(), "temperature": pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), "uniform": torch.rand(rows, generator=gen, device=DEV),
             "top_k": pick([0, 1, 20, 50, 200, 1000]).to(torch.int32) if "k" in case["cut"] else None, "top_p": pick([0.5, 0.8, 0.9, 0.95, 1.0]) if "p" in case["cut"] else None,
             "min_p": pick([0.0, 0.01, 0.05, 0.1]) if "m" in case["cut"] else None, "token": torch.zeros(rows, dtype=torch.int32, device=DEV), "logprob": torch.zeros(rows, device=DEV)}
        return {"case": case, **s}
    old, add = _lengths(case)
    block, seqs = case["block"], case["seqs"]
    if case["op"] == "plan":
        # the pool: blocks in use by the tables, the rest in the ring of free ones
        short = max(0, sum(_up(o + max(a, 0), block) - _up(o, block) for o, a in zip(old, add)))
        table, blocks = _pool(gen, old, [0] * seqs, block, spare=short + 64)
        width = max(table.shape[1], max(_up(o + max(a, 0), block) for o, a in zip(old, add))) + 3
        table = torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1).contiguous()
        used = torch.zeros(blocks + 1, dtype=torch.bool, device=DEV)
        used[torch.where(table < 0, blocks, table).long()] = True
        free = torch.nonzero(~used[:blocks])[:, 0].to(torch.int32)
        free = free[torch.randperm(free.numel(), generator=gen, device=DEV)]
        head = int(seed) % blocks
        ring = torch.full((blocks,), -1, dtype=torch.int32, device=DEV)
        ring[(head + torch.arange(free.numel(), device=DEV)) % blocks] = free
        rows = _up(sum(max(a, 0) for a in add) + 1, 64) * 64  # a padded step
        new = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
        return {"case": case, "ctx": i32(old), "new": i32(add), "table": table, "ring": ring, "state": i32([head, free.numel()]), "state_out": new(2), "next_len": new(seqs),
                "kv_len": new(seqs), "start": new(seqs + 1), "positions": new(rows), "slots": new(rows), "status": new(seqs)}
    table, blocks = _pool(gen, old, add, block, spare=5)
    cache = _cache(gen, blocks, case["kvh"], block, case["dim"])
    total = max(1, sum(add))
    start = i32(np.concatenate([[0], np.cumsum(add)]).tolist())
    t = torch.arange(total, device=DEV)
    s = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=seqs - 1)
    pos = i32(old)[s] + t - start[s]
    dtype = torch.float32 if case["f32"] else torch.float16
    qh, kvh, dim = case["qh"], case["kvh"], case["dim"]
    if case["op"] == "append":
        # the activations as a QKV projection leaves them, some channels of the keys larger than others
        x = torch.randn(total, qh + 2 * kvh, dim, generator=gen, device=DEV)
        x[:, qh:qh + kvh] *= 1 + 4 * (torch.rand(kvh, dim, generator=gen, device=DEV) < 0.05)
        slots = table[s, (pos // block).long()] * block + pos % block
        slots = torch.where(t < sum(add), slots, -1).to(torch.int32)
        f = _frequencies(case["rot"])
        angle = torch.arange(max(o + a for o, a in zip(old, add)) + 1, dtype=torch.float64, device=DEV)[:, None] * torch.from_numpy(f).to(DEV)
        # what the step's blocks hold afterwards is read back: their slots, in order
        touched = [np.arange(o // block * block, o + a) for o, a in zip(old, add)]
        whose = torch.from_numpy(np.concatenate([np.full(len(p) if a else 0, i) for i, (p, a) in enumerate(zip(touched, add))] + [np.zeros(0, np.int64)]).astype(np.int64)).to(DEV)
        where = torch.from_numpy(np.concatenate([p if a else p[:0] for p, a in zip(touched, add)] + [np.zeros(0, np.int64)]).astype(np.int64)).to(DEV)
        seen = (table[whose, where // block] * block + where % block).to(torch.int32)
        return {"case": case, "qkv": x.to(dtype), "positions": pos.to(torch.int32), "slots": slots, "rope": torch.stack([angle.cos(), angle.sin()], -1).float().contiguous(), **cache,
                "q_out": torch.zeros(total, qh, dim, dtype=dtype, device=DEV), "seen": seen, "k_out": torch.zeros(seen.numel(), kvh, dim, dtype=torch.float16, device=DEV),
                "v_out": torch.zeros(seen.numel(), kvh, dim, dtype=torch.float16, device=DEV)}
    rows = total + 3  # a few rows of padding behind the last sequence
    q = (torch.randn(rows, qh, dim, generator=gen, device=DEV) * 2).to(dtype)
    return {"case": case, "q": q, "y": torch.full((rows, qh, dim), 2.0 ** -8, dtype=dtype, device=DEV), "table": table, "start": start, "kv_len": i32([o + a for o, a in zip(old, add)]),
            "most": max(add), **cache}


# ------------------------------------------------------------------ the plain forms

def _plan(s):
    block, seqs, width = s["case"]["block"], s["case"]["seqs"], s["table"].shape[1]
    pool, rows = s["ring"].numel(), s["slots"].numel()
    ctx, new, table, head, count = s["ctx"].long(), s["new"].long(), s["table"], s["state"][0].long(), s["state"][1].long()
    bad = (ctx < 0) | (new < -1) | ((ctx + block - 1) // block > width)
    add = torch.where(bad, 0, new.clamp(min=0))
    end = torch.cumsum(add, 0)
    have, want = (ctx.clamp(min=0) + block - 1) // block, (ctx + add + block - 1) // block
    status = torch.where(bad, 4, torch.where(end > rows, 3, torch.where(want > width, 2, 0)))
    status = torch.where(add > 0, status, torch.where(bad, 4, 0))
    ask = torch.where((add > 0) & (status == 0), want - have, 0)
    upto = torch.cumsum(ask, 0)
    status = torch.where((ask > 0) & (upto > count), 1, status)
    fine = status == 0
    taken = torch.where((ask > 0) & fine, upto, 0).max()
    col = torch.arange(width, device=DEV)
    fresh = (col >= have[:, None]) & (col < want[:, None]) & ((ask > 0) & fine)[:, None]
    table = torch.where(fresh, s["ring"][(head + (upto - ask)[:, None] + col - have[:, None]) % pool], table)
    gone = (new == -1) & ~bad
    give = torch.where(gone, have, 0)
    at = (head + count + torch.cumsum(give, 0) - give)[:, None] + col
    ring = torch.cat([s["ring"], s["ring"][:1]])
    ring[torch.where(gone[:, None] & (col < have[:, None]), at % pool, pool)] = table
    start = torch.cat([end.new_zeros(1), end]).clamp(max=rows)
    t = torch.arange(rows, device=DEV)
    w = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=seqs - 1)
    live = t < start[-1]
    pos = torch.where(live, ctx[w] + t - start[w], 0)
    b = table[w, (pos // block).clamp(max=width - 1)].long()
    slots = torch.where(live & fine[w] & (b >= 0) & (b < pool), b * block + pos % block, -1)
    i = torch.int32
    return {"table": table, "ring": ring[:pool], "state": torch.stack([(head + taken) % pool, count - taken + give.sum()]).to(i), "start": start.to(i), "positions": pos.to(i), "slots": slots.to(i),
            "status": status.to(i), "kv_len": torch.where(fine & ~gone, ctx + add, 0).to(i), "next_len": torch.where(gone, 0, torch.where(fine, ctx + add, ctx)).to(i)}


def _rotate(x, rope, positions, pairs):
    x = x.float()
    n = rope.shape[1]
    cos, sin = rope[positions.long(), None].unbind(-1)
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1), x[..., 2 * n:]], -1)


def _store(codes, scale, x, slots):
    """x [tokens, heads, dim] at `slots` of codes [blocks, heads, tokens of a block, dim]: a block's scale grows to the
    smallest power of two that holds the new rows' largest value in 127 steps, what the block held is rounded to it."""
    blocks, heads, size, dim = codes.shape
    live = slots >= 0
    block, at = torch.where(live, slots // size, blocks).long(), (slots % size).long()
    most = torch.zeros(blocks + 1, heads, device=DEV).index_reduce_(0, block, x.abs().amax(-1), "amax")[:blocks]
    first = torch.full((blocks + 1,), size, dtype=torch.long, device=DEV).index_reduce_(0, block, at, "amin")[:blocks]
    m, e = torch.frexp(most)
    need = torch.where(most > 0, torch.ldexp(torch.ones_like(m), e - torch.where(m <= 127 / 128, 7, 6)), 2.0 ** -126)
    new = torch.where((first == size)[:, None], scale, torch.where((first == 0)[:, None], need, torch.maximum(scale, need)))
    kept = torch.arange(size, device=DEV) < first[:, None]
    codes = torch.where(kept[:, None, :, None], (codes * (scale / new)[..., None, None]).round().to(torch.int8), codes)
    value = (x / new[block.clamp(max=blocks - 1)][..., None]).round().clamp(-127, 127).to(torch.int8)
    codes = torch.cat([codes, codes[:1]])
    codes[block, :, at] = value
    return codes[:blocks], new


def _append(s):
    c = s["case"]
    q, k, v = s["qkv"].split([c["qh"], c["kvh"], c["kvh"]], 1)
    got = {"q": _rotate(q, s["rope"], s["positions"], c["pairs"]).to(q.dtype)}
    k, v = _rotate(k, s["rope"], s["positions"], c["pairs"]), v.float()
    block, at = (s["seen"] // c["block"]).long(), (s["seen"] % c["block"]).long()
    for name, x in (("k", k), ("v", v)):
        codes, scale = _store(s[name], s[name + "_scale"], x, s["slots"])
        got[name] = (codes[block, :, at].float() * scale[block][..., None]).half()
    return got


def _attn(s):
    c = s["case"]
    block, heads, group, most = c["block"], c["kvh"], c["qh"] // c["kvh"], max(1, s["most"])
    start, length, rows = s["start"].long(), s["kv_len"].long(), s["q"].shape[0]
    used = s["table"].clamp(min=0).long()
    i = torch.arange(most, device=DEV)
    row = (start[:-1, None] + i).clamp(max=rows - 1)
    q = s["q"][row].float().unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [sequence, head, group * token, dim]

    def cached(name):
        x = s[name][used].float() * s[name + "_scale"][used][..., None, None]
        return x.permute(0, 2, 1, 3, 4).flatten(2, 3)

    score = (q @ cached("k").transpose(-1, -2) / math.sqrt(c["dim"])).unflatten(2, (group, most))
    key = torch.arange(score.shape[-1], device=DEV)
    last = (length - (start[1:] - start[:-1]))[:, None] + i
    seen = (key <= last[..., None]) & (key < length[:, None, None])
    if c["window"]:
        seen = seen & (key > last[..., None] - c["window"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ cached("v")).unflatten(2, (group, most)) / torch.where(total == 0, 1, total)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [sequence, token, query head, dim]
    t = torch.arange(rows, device=DEV)
    w = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=c["seqs"] - 1)
    live = t < start[-1]
    return torch.where(live[:, None, None], out[w, torch.where(live, t - start[w], 0)].to(s["y"].dtype), s["y"])


def _sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1))
    rank = torch.arange(vocab, device=DEV)
    keep = torch.where(t > 0, rank < vocab, rank < 1)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep = keep & ((k <= 0) | (rank < k))
    w = torch.where(keep, w, 0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        w = torch.where((p >= 1) | (rank == 0) | (torch.cumsum(w, 1) - w < p * w.sum(1, keepdim=True)), w, 0)
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"].double()[:, None], w, 0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # in the vocabulary's order
    upto = torch.cumsum(w, 1)
    token = (upto <= s["uniform"].double()[:, None] * upto[:, -1:]).sum(1, keepdim=True).clamp(max=vocab - 1)
    return {"token": token[:, 0].to(torch.int32), "logprob": torch.log(w.gather(1, token) / upto[:, -1:])[:, 0].float()}


def run(s):
    op, c = s["case"]["op"], s["case"]
    if not own:
        return {"plan": _plan, "append": _append, "attn": _attn, "sample": _sample}[op](s)
    from ztensor_b200 import kernels as K
    if op == "plan":
        K.kv_plan(s["ctx"], s["new"], s["table"], s["ring"], s["state"], s["state_out"], s["next_len"], s["kv_len"], s["start"], s["positions"], s["slots"], s["status"], c["block"])
        return {"table": s["table"], "ring": s["ring"], "state": s["state_out"], "start": s["start"], "positions": s["positions"], "slots": s["slots"], "status": s["status"], "kv_len": s["kv_len"],
                "next_len": s["next_len"]}
    if op == "sample":
        K.sample(s["logits"], s["uniform"], s["token"], s["logprob"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"token": s["token"], "logprob": s["logprob"]}
    if "cache" not in s:  # a program makes these once, beside its buffers
        s["cache"] = K.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if op == "append":
            s["q"], s["new_k"], s["new_v"] = s["qkv"].split([c["qh"], c["kvh"], c["kvh"]], 1)
        else:
            s["workspace"] = torch.empty(K.attn_q8_workspace_bytes(s["q"].shape[0], c["seqs"], s["most"], c["qh"], c["kvh"], c["dim"]), dtype=torch.uint8, device=DEV)
    if op == "append":
        K.rope_append_q8(s["q"], s["new_k"], s["new_v"], s["q_out"], s["slots"], s["cache"], s["rope"], s["positions"], K.ROPE_PAIRS if c["pairs"] else 0)
        K.kv_read_q8(s["cache"], s["seen"], s["k_out"], s["v_out"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    K.attn_q8(s["q"], s["y"], s["start"], s["kv_len"], s["table"], s["cache"], s["workspace"], s["most"], 1 / math.sqrt(c["dim"]), c["window"])
    return s["y"]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["f32"] else 2) + case["rows"] * 28, "flops": 3 * n}
    old, add = _lengths(case)
    if case["op"] == "plan":
        tokens = sum(max(a, 0) for a in add)
        moved = sum(_up(o + a, case["block"]) - _up(o, case["block"]) if a > 0 else _up(o, case["block"]) if a < 0 else 0 for o, a in zip(old, add))
        return {"bytes": 4 * (6 * case["seqs"] + 2 * tokens + 2 * moved + 4), "flops": 4 * tokens}
    e, dim, kvh, qh = 4 if case["f32"] else 2, case["dim"], case["kvh"], case["qh"]
    if case["op"] == "append":
        tokens, seen = sum(add), sum((o + a) - o // case["block"] * case["block"] for o, a in zip(old, add) if a)
        return {"bytes": tokens * ((2 * qh + 2 * kvh) * dim * e + 2 * kvh * dim + case["rot"] * 4 + 8) + seen * (2 * kvh * dim * 3 + 4), "flops": tokens * (3 * (qh + kvh) * case["rot"] + 3 * 2 * kvh * dim)}
    read, pairs = 0, 0
    for o, a in zip(old, add):
        w = case["window"] or (o + a)
        first = max(0, o + 1 - w)
        read += (o + a - first) if a else 0
        full = max(0, min(a, w - o))  # queries whose window reaches back to the first key
        pairs += full * o + full * (full + 1) // 2 + (a - full) * w
    return {"bytes": read * kvh * (2 * dim + 8 / case["block"]) + 2 * sum(add) * qh * dim * e, "flops": 4 * pairs * qh * dim}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_append(s) if case["op"] == "append" else _exact_attn(s)


def _exact_sample(s):
    get = lambda name: None if s[name] is None else s[name].cpu().numpy().astype(np.float64)  # noqa: E731
    x, t, k, p, m, u = (get(n) for n in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform"))
    tokens, logs = [], []
    for r in range(x.shape[0]):
        order = np.lexsort((np.arange(x.shape[1]), -x[r]))
        if t[r] <= 0:
            order, w = order[:1], np.ones(1)
        else:
            if k is not None and k[r] > 0:
                order = order[:int(k[r])]
            w = np.exp((x[r, order] - x[r, order[0]]) / t[r])
        if p is not None and p[r] < 1:
            n = max(1, int(np.sum(np.concatenate([[0.0], np.cumsum(w)[:-1]]) < p[r] * w.sum())))
            order, w = order[:n], w[:n]
        if m is not None:
            order, w = order[w >= m[r]], w[w >= m[r]]
        by = np.argsort(order)
        order, w = order[by], w[by]
        upto = np.cumsum(w)
        i = min(int(np.searchsorted(upto, u[r] * upto[-1], side="right")), len(w) - 1)
        tokens.append(order[i])
        logs.append(math.log(w[i] / upto[-1]))
    return {"token": np.array(tokens, np.int32), "logprob": np.array(logs)}


def _exact_append(s):
    c = s["case"]
    old, add = _lengths(c)
    dim, n, size = c["dim"], c["rot"] // 2, c["block"]
    x = s["qkv"].double()
    turn = torch.exp(1j * s["positions"].double()[:, None] * torch.from_numpy(_frequencies(c["rot"])).to(DEV))[:, None]
    part = torch.stack([torch.arange(n) * 2, torch.arange(n) * 2 + 1] if c["pairs"] else [torch.arange(n), torch.arange(n) + n]).to(DEV)
    z = torch.complex(x[:, :c["qh"] + c["kvh"], part[0]], x[:, :c["qh"] + c["kvh"], part[1]]) * turn
    x[:, :c["qh"] + c["kvh"], part[0]], x[:, :c["qh"] + c["kvh"], part[1]] = z.real, z.imag
    out = {"q": x[:, :c["qh"]], "k": [], "v": []}
    row = 0
    slots, at = s["seen"].cpu().numpy(), 0
    for o, a in zip(old, add):
        for b in range(o // size, _up(o + a, size) if a else 0):
            first, upto = max(o, b * size), min(o + a, (b + 1) * size)
            keep, block = first - b * size, int(slots[at]) // size
            for name, h in (("k", c["qh"]), ("v", c["qh"] + c["kvh"])):
                y = x[row + first - o:row + upto - o, h:h + c["kvh"]].transpose(0, 1)
                most = y.abs().amax((1, 2))
                need = torch.where(most > 0, torch.exp2(torch.ceil(torch.log2(most / 127))), 2.0 ** -126)
                had = s[name + "_scale"][block].double()
                scale = torch.maximum(had, need) if keep else need
                held = torch.round(s[name][block, :, :keep].double() * (had / scale)[:, None, None])
                fresh = torch.round(y / scale[:, None, None])
                out[name].append((torch.cat([held, fresh], 1) * scale[:, None, None]).transpose(0, 1))
            at += keep + upto - first
        row += a
    return {"q": out["q"], "k": torch.cat(out["k"]), "v": torch.cat(out["v"])}


def _exact_attn(s):
    c = s["case"]
    old, add = _lengths(c)
    group, row = c["qh"] // c["kvh"], 0
    y = s["y"].double()
    for b, (o, a) in enumerate(zip(old, add)):
        if not a:
            continue
        n = o + a
        blocks = s["table"][b, :_up(n, c["block"])].long()
        position = torch.arange(n, device=DEV)
        for h in range(c["kvh"]):
            k, v = ((s[name][blocks, h].double() * s[name + "_scale"][blocks, h].double()[:, None, None]).reshape(-1, c["dim"])[:n] for name in ("k", "v"))
            gap = (o + torch.arange(a, device=DEV))[:, None] - position
            hidden = (gap < 0) | (gap >= (c["window"] or n + 1))
            for g in range(h * group, (h + 1) * group):
                score = s["q"][row:row + a, g].double() @ k.T / c["dim"] ** 0.5
                y[row:row + a, g] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
        row += a
    return y
