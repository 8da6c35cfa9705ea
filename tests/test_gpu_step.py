"""The decode-step operators (plan, rotary positions, 8-bit cache, attention, sampling) against 64-bit references."""
import math

import numpy as np
import pytest
import torch

from tests import step_ref as R
from tests import util as U
from ztensor_b200 import _lib
from ztensor_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF16, HALF32 = 2.0 ** -11, 2.0 ** -24          # half steps of fp16 and fp32


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV) if dtype is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def host(t):
    return t.float().cpu().numpy().astype(np.float64) if t.is_floating_point() else t.cpu().numpy()


def no_error():
    assert K.device_error() == 0


# ------------------------------------------------------------------ plan

def plan_case(rng, n, block, shape):
    """Lengths, a table holding the cached blocks and a ring holding the free ones."""
    ctx = rng.integers(0, 6 * block, n)
    new = rng.choice([0, 1, 1, 1, 3, 2 * block + 5], n)
    if shape != "plain":
        new[rng.random(n) < 0.3] = -1
    have = -(-ctx // block)
    width = int(max(have.max(), (-(-(ctx + np.maximum(new, 0)) // block)).max())) + (0 if shape == "narrow" else 2)
    width = max(1, width - 2 if shape == "narrow" else width)
    if shape == "narrow":
        ctx = np.minimum(ctx, width * block)
        have = -(-ctx // block)
    ask = int(np.where(new > 0, -(-(ctx + np.maximum(new, 0)) // block) - have, 0).sum())
    free = ask // 2 if shape == "short" else ask + 3
    pool = int(have.sum()) + free
    order = rng.permutation(max(pool, 1)).astype(np.int32)
    table = np.full((n, width), -7, np.int32)
    at = 0
    for b in range(n):
        table[b, :have[b]] = order[at:at + have[b]]
        at += have[b]
    pool = max(pool, 1)
    head = int(rng.integers(0, pool))
    ring = np.full(pool, -1, np.int32)
    ring[(head + np.arange(free)) % pool] = order[at:at + free]
    if shape == "bad":
        ctx[0], new[-1] = -4, -9
        ctx[n // 2] = width * block + 1
    rows = max(1, int(np.maximum(new, 0).sum()) + (-2 if shape == "rows" else 5))
    return ctx.astype(np.int32), new.astype(np.int32), table, ring, np.array([head, free], np.int32), rows


@pytest.mark.parametrize("shape", ["plain", "release", "short", "narrow", "rows", "bad"])
@pytest.mark.parametrize("n,block", [(1, 16), (7, 32), (300, 64), (1500, 16), (4096, 128)])
def test_plan(n, block, shape):
    ctx, new, table, ring, state, rows = plan_case(U.seeded(n + block), n, block, shape)
    want = R.kv_plan(ctx, new, table, ring, state, block, rows)
    for alias in (False, True):                  # lengths and ring state in place, or not
        t = {"block_table": dev(table), "ring": dev(ring)}
        c, s = dev(ctx), dev(state)
        for name, shape_ in (("kv_len", n), ("query_start", n + 1), ("positions", rows), ("slots", rows), ("status", n)):
            t[name] = torch.full((shape_,), -77, dtype=torch.int32, device=DEV)
        t["next_len"], t["ring_state_out"] = (c, s) if alias else (torch.empty_like(c), torch.empty_like(s))
        K.kv_plan(c, dev(new), t["block_table"], t["ring"], s, t["ring_state_out"], t["next_len"], t["kv_len"], t["query_start"], t["positions"], t["slots"], t["status"], block)
        for name, w in want.items():
            assert np.array_equal(host(t[name]), w), (name, alias)
    no_error()


# ------------------------------------------------------------------ rotary positions

SCALINGS = [("none", {}), ("linear", dict(factor=4.0)), ("by_turns", dict(factor=8.0, turns_low=1.0, turns_high=4.0, original_positions=8192)),
            ("by_dim", dict(factor=16.0, turns_low=1.0, turns_high=32.0, original_positions=4096, magnitude=1.277))]


@pytest.mark.parametrize("scaling,kw", SCALINGS)
@pytest.mark.parametrize("first,rows", [(0, 1), (5, 33), (1 << 20, 40), ((1 << 31) - 20, 19)])
def test_rope_table(scaling, kw, first, rows):
    for rot, base in ((16, 10000.0), (128, 500000.0), (256, 1e6)):
        got = host(K.rope_table(rows, rot, base, first=first, scaling=scaling, **kw))
        f = R.frequencies(rot, base, scaling, kw.get("factor", 1.0), kw.get("turns_low", 1.0), kw.get("turns_high", 4.0), kw.get("original_positions", 0.0))
        angle = (first + np.arange(rows, dtype=np.float64))[:, None] * f
        want = np.stack([np.cos(angle), np.sin(angle)], -1) * kw.get("magnitude", 1.0)
        # one rounding to fp32, and the angle's own rounding in 64 bits (its frequency within a few steps of 2^-53)
        assert (np.abs(got - want) <= 2 * HALF32 + angle[..., None] * 2.0 ** -50).all()
    no_error()


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("x32,y32", [(False, False), (True, True), (False, True), (True, False)])
@pytest.mark.parametrize("tokens,heads,dim,rot,layout", [(1, 1, 16, 16, "packed"), (3, 5, 64, 32, "packed"), (37, 8, 128, 128, "qkv"), (130, 7, 80, 48, "odd"), (17, 3, 256, 256, "heads_first"),
                                                         (16, 64, 128, 128, "in_place")])
def test_rope(pairs, x32, y32, tokens, heads, dim, rot, layout):
    if layout == "in_place" and x32 != y32:
        pytest.skip("one type in place")
    rng = U.seeded(tokens + dim)
    table = K.rope_table(500, rot, 10000.0)
    pos = rng.integers(0, 500, tokens).astype(np.int32)
    a = rng.standard_normal((tokens, heads, dim))
    xt, yt = torch.float32 if x32 else torch.float16, torch.float32 if y32 else torch.float16
    if layout == "qkv":                          # a slice of a wider row
        wide = torch.zeros(tokens, heads + 3, dim, dtype=xt, device=DEV)
        x = wide[:, 2:2 + heads]
    elif layout == "odd":                        # rows that start on odd elements
        x = torch.zeros(tokens * (heads * dim + 1) + 1, dtype=xt, device=DEV)[1:].as_strided((tokens, heads, dim), (heads * dim + 1, dim, 1))
    elif layout == "heads_first":
        x = torch.zeros(heads, tokens, dim, dtype=xt, device=DEV).transpose(0, 1)
    else:
        x = torch.zeros(tokens, heads, dim, dtype=xt, device=DEV)
    x.copy_(dev(a))
    ref = R.rope(host(x), host(table), pos, pairs)
    mag = np.abs(host(x)).max() * 2
    y = x if layout == "in_place" else torch.full((tokens, heads, dim), math.nan, dtype=yt, device=DEV)
    K.rope(x, y, table, dev(pos), K.ROPE_PAIRS if pairs else 0)
    # two products and a sum in fp32, then the output's half step (fp16: 2^-25 below the normal range)
    tol = 3 * HALF32 * mag + (0 if y32 else HALF16 * np.abs(ref) + 2.0 ** -25)
    assert (np.abs(host(y) - ref) <= tol).all()
    no_error()


def test_rope_position_outside_the_table():
    table = K.rope_table(10, 32, 10000.0)
    x = torch.ones(4, 2, 64, device=DEV)
    y = torch.zeros_like(x)
    K.rope(x, y, table, dev(np.array([0, 10, -1, 9], np.int32)))
    assert torch.isnan(y[1:3, :, :32]).all() and not torch.isnan(y[[0, 3]]).any() and (y[..., 32:] == 1).all()
    assert K.device_error() == 6 and K.device_error() == 0


# ------------------------------------------------------------------ cache

def random_cache(rng, blocks, heads, size, dim, interleaved=False):
    """A cache with arbitrary codes and scales; interleaved: k and v blocks alternate in one allocation."""
    if interleaved:
        both = torch.empty(blocks, 2, heads, size, dim, dtype=torch.int8, device=DEV)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.empty(blocks, heads, size, dim, dtype=torch.int8, device=DEV) for _ in range(2))
    for t in (k, v):
        t.copy_(dev(rng.integers(-127, 128, t.shape).astype(np.int8)))
    scales = [dev(np.exp2(rng.integers(-9, -4, (blocks, heads))).astype(np.float32)) for _ in range(2)]
    return K.KvCache(k, v, *scales)


@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("tokens,heads,qh,size,dim,rot,layout", [(1, 1, 1, 16, 16, 16, "decode"), (40, 2, 6, 16, 64, 64, "decode"), (200, 3, 21, 32, 128, 64, "prompt"), (333, 1, 4, 128, 256, 256, "prompt"),
                                                                 (97, 2, 0, 64, 80, 0, "mixed"), (64, 8, 64, 16, 128, 128, "mixed")])
def test_append(x32, tokens, heads, qh, size, dim, rot, layout):
    rng = U.seeded(tokens + size)
    blocks = tokens + 3 if layout == "decode" else 2 * tokens // size + 8
    cache = random_cache(rng, blocks, heads, size, dim, interleaved=layout == "mixed")
    k0, v0, ks0, vs0 = (t.cpu().numpy() for t in cache.tensors)
    order = rng.permutation(blocks)
    slots = np.full(tokens, -1, np.int64)
    if layout == "decode":                       # one token per block, anywhere in it
        slots[:] = order[:tokens] * size + rng.integers(0, size, tokens)
    else:                                        # runs that begin and end inside blocks, with skipped rows between
        t = b = 0
        while t < tokens:
            n = min(int(rng.integers(1, 3 * size)), tokens - t)
            off = int(rng.integers(0, size))
            for i in range(n):
                if off == size:
                    off, b = 0, b + 1
                if b < blocks:
                    slots[t + i] = order[b] * size + off
                off += 1
            b += 1
            t += n + (2 if layout == "mixed" else 0)
    slots = slots.astype(np.int32)
    dtype = torch.float32 if x32 else torch.float16
    x = torch.zeros(tokens, qh + 2 * heads, dim, dtype=dtype, device=DEV)
    a = rng.standard_normal(x.shape) * np.exp2(rng.integers(-4, 5, (tokens, qh + 2 * heads, 1)))
    if tokens > 30:
        a[5:9] = 0                               # rows without any size
    x.copy_(dev(a))
    q, k, v = x.split([qh, heads, heads], 1)
    table = K.rope_table(300, rot, 10000.0) if rot else None
    pos = rng.integers(0, 300, tokens).astype(np.int32)
    q_out = torch.full((tokens, qh, dim), math.nan, dtype=dtype, device=DEV) if qh else None
    K.rope_append_q8(q if qh else None, k, v, q_out, dev(slots), cache, table, dev(pos) if rot else None, K.ROPE_PAIRS if layout == "mixed" else 0)
    turn = lambda t: R.rope(host(t), host(table), pos, layout == "mixed") if rot else host(t)  # noqa: E731
    if qh:
        ref = turn(q)
        assert (np.abs(host(q_out) - ref) <= 3 * HALF32 * 2 * np.abs(host(q)).max() + (0 if x32 else HALF16 * np.abs(ref) + 2.0 ** -25)).all()
    for name, rows, codes0, scale0, codes, scale in (("k", turn(k), k0, ks0, cache.tensors[0], cache.tensors[2]), ("v", host(v), v0, vs0, cache.tensors[1], cache.tensors[3])):
        want, s = R.append(codes0, scale0, rows, slots)
        assert np.array_equal(host(scale), s.astype(np.float64)), name
        got = host(codes)
        # the rotation's fp32 rounding can move a value over the border between two codes, never further
        differ = got != want
        assert not differ.any() if name == "v" or not rot else (np.abs(got.astype(int) - want).max() <= 1 and differ.mean() < 1e-4), name
    # reading back: the codes times their scale, one rounding
    seen = dev(np.concatenate([slots, [-1, blocks * size, slots.max()]]).astype(np.int32))
    for t in (torch.float16, torch.float32):
        ko, vo = (torch.full((len(seen), heads, dim), 7.0, dtype=t, device=DEV) for _ in range(2))
        K.kv_read_q8(cache, seen, ko, vo)
        for out, codes, scale in ((ko, cache.tensors[0], cache.tensors[2]), (vo, cache.tensors[1], cache.tensors[3])):
            c, s, out = host(codes).astype(np.float64), host(scale), host(out)
            for i, slot in enumerate(seen.tolist()):
                if 0 <= slot < blocks * size:
                    want = c[slot // size, :, slot % size] * s[slot // size][:, None]
                    assert np.array_equal(out[i], want if t is torch.float32 else want.astype(np.float16).astype(np.float64))
                else:
                    assert (out[i] == 7).all()
    no_error()


@pytest.mark.parametrize("x32", [False, True])
def test_append_rotates_queries_into_the_other_type(x32):
    rng = U.seeded(16)
    cache, table = random_cache(rng, 40, 2, 16, 64), K.rope_table(100, 64, 10000.0)
    x = dev(rng.standard_normal((21, 8, 64)), torch.float32 if x32 else torch.float16)
    q, k, v = x.split([4, 2, 2], 1)
    out = torch.zeros(21, 4, 64, dtype=torch.float16 if x32 else torch.float32, device=DEV)
    pos = rng.integers(0, 100, 21).astype(np.int32)
    K.rope_append_q8(q, k, v, out, dev(np.arange(21, dtype=np.int32) * 16), cache, table, dev(pos))
    ref = R.rope(host(q), host(table), pos, False)
    assert (np.abs(host(out) - ref) <= 3 * HALF32 * 2 * np.abs(host(q)).max() + (HALF16 * np.abs(ref) + 2.0 ** -25 if x32 else 0)).all()
    no_error()


def test_append_grows_a_block_step_by_step():
    """One token per step into one block, each larger than all before: every step rounds the old rows once."""
    cache = K.KvCache.empty(2, 1, 16, 64)
    rng = U.seeded(3)
    codes, scale = np.zeros((2, 1, 16, 64), np.int8), np.zeros((2, 1), np.float32)
    for t in range(16):
        x = dev(rng.standard_normal((1, 1, 64)) * 1.7 ** t, torch.float16)
        slots = np.array([16 + t], np.int32)
        K.rope_append_q8(None, x, x, None, dev(slots), cache)
        codes, scale = R.append(codes, scale, host(x), slots)
        assert np.array_equal(host(cache.tensors[1])[1, :, :t + 1], codes[1, :, :t + 1]) and np.array_equal(host(cache.tensors[3])[1], scale[1])
    no_error()


def test_append_not_finite_until_the_block_begins_anew():
    cache = K.KvCache.empty(1, 2, 16, 64)
    one = torch.ones(1, 2, 64, device=DEV)
    for slot, bad in ((0, None), (1, math.nan), (2, None), (0, math.inf), (0, None)):
        x = one.clone()
        if bad is not None:
            x[0, 1, 5] = bad
        K.rope_append_q8(None, one, x, None, dev(np.array([slot], np.int32)), cache)
        nan = torch.isnan(cache.tensors[3])[0].tolist()
        assert not torch.isnan(cache.tensors[2]).any() and nan == [False, bad is not None or slot == 2]
    no_error()


@pytest.mark.parametrize("slots", [[16, 18], [5, 4], [3, 3], [1 << 20, 2]])
def test_append_rows_out_of_order_are_skipped(slots):
    cache = random_cache(U.seeded(1), 4, 1, 16, 64)
    before = [t.clone() for t in cache.tensors]
    x = torch.ones(2, 1, 64, device=DEV)
    K.rope_append_q8(None, x, x, None, dev(np.array(slots, np.int32)), cache)
    good = [s for i, s in enumerate(slots) if s < 64 and (i == 0 or slots[0] >= 64)]
    codes, scale = R.append(before[0].cpu().numpy(), before[2].cpu().numpy(), np.ones((1, 1, 64)), good)
    assert np.array_equal(host(cache.tensors[0]), codes) and np.array_equal(host(cache.tensors[2]), scale.astype(np.float64))
    assert K.device_error() == 5 and K.device_error() == 0


# ------------------------------------------------------------------ attention

def attn_case(rng, lens, heads, group, size, dim, dtype, layout="packed", spare=3):
    """lens: (tokens in the cache, new tokens) of each sequence."""
    need = [-(-n // size) for n, _ in lens]
    blocks = sum(need) + spare
    cache = random_cache(rng, blocks, heads, size, dim, interleaved=layout == "heads_first")
    order = rng.permutation(blocks).astype(np.int32)
    table = np.full((len(lens), max(need + [1]) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum([a for _, a in lens])]).astype(np.int32)
    rows, qh = int(start[-1]) + 2, heads * group
    if layout == "heads_first":
        q, y = (torch.zeros(qh, rows, dim, dtype=dtype, device=DEV).transpose(0, 1) for _ in range(2))
    elif layout == "odd":
        q, y = (torch.zeros(rows * (qh * dim + 3) + 1, dtype=dtype, device=DEV)[1:].as_strided((rows, qh, dim), (qh * dim + 3, dim, 1)) for _ in range(2))
    else:
        q, y = (torch.zeros(rows, qh, dim, dtype=dtype, device=DEV) for _ in range(2))
    q.copy_(dev(rng.standard_normal((rows, qh, dim)) * 1.5))
    y.fill_(0.5)
    return cache, dev(table), dev(start), dev(np.array([n for n, _ in lens], np.int32)), q, y


def attn_check(lens, cache, table, start, q, y, scale, window, f32):
    k, v, ks, vs = (host(t).astype(np.float64) for t in cache.tensors)
    group = q.shape[1] // cache.kv_heads
    got, qh, table = host(y), host(q), table.cpu().numpy()
    row = 0
    for b, (n, a) in enumerate(lens):
        blocks = table[b, :-(-n // cache.block_size)]
        for h in range(cache.kv_heads):
            kk = (k[blocks, h] * ks[blocks, h][:, None, None]).reshape(-1, cache.head_dim)[:n]
            vv = (v[blocks, h] * vs[blocks, h][:, None, None]).reshape(-1, cache.head_dim)[:n]
            for g in range(h * group, (h + 1) * group):
                ref, mean, size, _ = R.attention(qh[row:row + a, g], kk, vv, n - a, scale, window)
                # scores: fp32 sums of exact products (q in one or two fp16 terms), D / 16 + 2 roundings of the running
                # sum; weights: the half step of fp16, or of two terms; sums and division in fp32; the output's half step.
                # A weight far below the largest ends at fp16's last step: weights times the V scale over a power of two, at
                # most the largest scale of the cache, are held times 2^4 (fp32: 2^12) and the last half step is 2^-25, so
                # each is off by up to 2^-29 (2^-37) of the largest, whose weight is at least 1 of the sum's parts
                ends = (2.0 ** -37 if f32 else 2.0 ** -29) * np.abs(vs).max() * np.abs(v[blocks, h]).reshape(-1, cache.head_dim)[:n].sum(0)
                term = 2.0 ** -22 if f32 else 0.0
                weight = (cache.head_dim / 16 + 2) * 2 * HALF32 * size + term * size + (4 * 2.0 ** -22 if f32 else HALF16) + 64 * HALF32
                tol = 2 * weight * mean + ends + (0 if f32 else HALF16 * np.abs(ref) + 2.0 ** -25) + 2.0 ** -40
                assert (np.abs(got[row:row + a, g] - ref) <= tol).all(), (b, g, float(np.max(np.abs(got[row:row + a, g] - ref) / tol)))
        row += a
    assert (got[row:] == 0.5).all()              # rows behind the last sequence


def attn_run(lens, heads, group, size, dim, f32=False, window=0, layout="packed", seed=0, scale=None, most=None):
    rng = U.seeded(seed)
    case = attn_case(rng, lens, heads, group, size, dim, torch.float32 if f32 else torch.float16, layout)
    cache, table, start, kv_len, q, y = case
    scale = scale if scale is not None else 1 / math.sqrt(dim)
    most = most or max(1, max(a for _, a in lens))
    ws = torch.full((K.attn_q8_workspace_bytes(q.shape[0], len(lens), most, q.shape[1], heads, dim) // 4,), math.nan, device=DEV)
    K.attn_q8(q, y, start, kv_len, table, cache, ws, most, scale, window)
    attn_check(lens, cache, table, start, q, y, scale, window, f32)
    no_error()
    return case, ws


ONE = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (200, 1), (1000, 1)]
FEW = [(5, 5), (40, 3), (0, 0), (64, 2), (129, 4), (300, 0), (33, 1)]
MANY = [(70, 70), (300, 45), (17, 16), (200, 1), (130, 64), (90, 33)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group,heads", [(1, 3), (4, 2), (8, 1), (7, 2), (16, 1), (3, 1)])
@pytest.mark.parametrize("lens", [ONE, FEW, MANY], ids=["one", "few", "many"])
def test_attn(dim, group, heads, lens):
    attn_run(lens, heads, group, 16 << (group % 4), dim, seed=dim + group)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("layout", ["packed", "odd", "heads_first"])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 100])
@pytest.mark.parametrize("lens", [ONE, FEW, MANY], ids=["one", "few", "many"])
def test_attn_windows_types_and_strides(f32, layout, window, lens):
    attn_run(lens, 2, 5, 32, 64 if window % 2 else 128, f32=f32, window=window, layout=layout, seed=window)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("x32,y32", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("lens", [ONE[2:6], FEW, MANY], ids=["one", "few", "many"])
def test_attn_types_apart(dim, x32, y32, lens):
    """Queries and outputs of different types; windows as large as an int holds."""
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 3, 16, dim, torch.float32 if x32 else torch.float16)
    y = torch.full(q.shape, 0.5, dtype=torch.float32 if y32 else torch.float16, device=DEV)
    most = max(a for _, a in lens)
    ws = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], len(lens), most, 6, 2, dim), dtype=torch.uint8, device=DEV)
    for window in (0, 2 ** 31 - 1, 17):
        K.attn_q8(q, y, start, kv_len, table, cache, ws, most, 0.1, window)
        attn_check(lens, cache, table, start, q, y, 0.1, min(window, 1 << 20), y32)
    no_error()


MIXED = [(300 + 7 * i, 1 if i % 3 else 30 + i) for i in range(40)]         # more heads than SMs: both kernels share the batch


@pytest.mark.parametrize("lens,heads,group,dim", [(MIXED, 4, 4, 64), (MIXED, 4, 3, 128), ([(20001, 1)], 8, 8, 128), ([(9000, 1), (3, 1), (5000, 1)], 1, 1, 64), ([(5000, 3)], 2, 4, 256), ([(3000, 260)], 2, 4, 128),
                                                  ([(700, 1)] * 90, 2, 8, 64)])
def test_attn_long(lens, heads, group, dim):
    attn_run(lens, heads, group, 64, dim, seed=len(lens))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 50])
def test_attn_scales_of_any_kind(new, dim):
    """Scales that are no powers of two, far apart, zero and negative: the append writes none of these, other writers may."""
    lens = [(300, new), (50 + new, new)]
    rng = U.seeded(13)
    cache, table, start, kv_len, q, y = attn_case(rng, lens, 2, 4, 16, dim, torch.float16)
    for t in cache.tensors[2:]:
        s = rng.uniform(0.5, 1.5, t.shape) * np.exp2(rng.integers(-16, -4, t.shape)) * rng.choice([1, 1, 1, -1, 0], t.shape)
        t.copy_(dev(s.astype(np.float32)))
    ws = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 2, new, 8, 2, dim), dtype=torch.uint8, device=DEV)
    for scale in (0.1, -0.1, 0.0):
        K.attn_q8(q, y, start, kv_len, table, cache, ws, new, scale)
        attn_check(lens, cache, table, start, q, y, scale, 0, False)
    no_error()


@pytest.mark.parametrize("new", [1, 3, 40])
def test_attn_rows_that_see_nothing_are_zero(new):
    """More rows than cached tokens: the first rows stand before position 0."""
    lens = [(2, new), (0, new), (50, new)]
    (cache, table, start, kv_len, q, y), ws = attn_run([(2, 2 if new > 1 else 1), (50, new)], 2, 4, 16, 64)
    rng = U.seeded(1)
    cache, table, start, kv_len, q, y = attn_case(rng, lens, 2, 4, 16, 64, torch.float16)
    K.attn_q8(q, y, start, kv_len, table, cache, torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 3, new, 8, 2, 64), dtype=torch.uint8, device=DEV), new, 0.125)
    attn_check(lens, cache, table, start, q, y, 0.125, 0, False)
    assert (y[new:2 * new] == 0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_attn_what_is_not_seen_does_not_count(new):
    """NaN scales of unseen blocks, garbage behind a sequence's end, blocks behind the table: none of it reaches a row."""
    lens = [(100, new), (37 + new, new)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(2), lens, 2, 4, 16, 128, torch.float16)
    used = set(table.cpu().numpy().ravel().tolist()) - {-1}
    for b in range(cache.blocks):
        if b not in used:
            cache.tensors[2][b] = math.nan
            cache.tensors[3][b] = math.inf
    window = 20                                  # the first blocks of the long sequence are out of every row's window
    first = (100 - new - window) // 16
    for b in range(max(first, 0)):
        cache.tensors[2][int(table[0, b])] = math.nan
        cache.tensors[3][int(table[0, b])] = math.nan
    ws = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 2, new, 8, 2, 128), dtype=torch.uint8, device=DEV)
    K.attn_q8(q, y, start, kv_len, table, cache, ws, new, 0.1, window)
    for t in cache.tensors[2:]:
        t.nan_to_num_(0, 0, 0)
    attn_check(lens, cache, table, start, q, y, 0.1, window, False)


@pytest.mark.parametrize("new", [3, 40])
@pytest.mark.parametrize("which", [2, 3])
def test_attn_a_nan_scale_reaches_the_rows_that_see_it(new, which):
    """The last block's scale is NaN: rows of its tokens become NaN, rows before them do not."""
    n = 64 + new
    cache, table, start, kv_len, q, y = attn_case(U.seeded(4), [(n, new)], 2, 4, 16, 64, torch.float16)
    cache.tensors[which][int(table[0, (n - 1) // 16]), 1] = math.nan
    ws = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 1, new, 8, 2, 64), dtype=torch.uint8, device=DEV)
    K.attn_q8(q, y, start, kv_len, table, cache, ws, new, 0.1)
    bad = torch.isnan(y[:new])
    sees = torch.arange(64, n, device=DEV) >= (n - 1) // 16 * 16
    assert not bad[:, :4].any() and torch.equal(bad[:, 4:].all(-1), sees[:, None].expand(-1, 4)) and torch.equal(bad[:, 4:].any(-1), bad[:, 4:].all(-1))


def test_attn_table_entries_outside_the_cache_are_hidden():
    for new in (1, 40):
        lens = [(16 * 6, new)]
        cache, table, start, kv_len, q, y = attn_case(U.seeded(5), lens, 1, 2, 16, 64, torch.float16)
        table[0, 1], table[0, 2] = -5, cache.blocks
        ws = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 1, new, 2, 1, 64), dtype=torch.uint8, device=DEV)
        K.attn_q8(q, y, start, kv_len, table, cache, ws, new, 0.1)
        assert K.device_error() == 7 and K.device_error() == 0
        k, v, ks, vs = (host(t).astype(np.float64) for t in cache.tensors)
        rows = [int(table[0, j // 16]) * 16 + j % 16 for j in range(96) if not 16 <= j < 48]
        kk, vv = (c.transpose(0, 2, 1, 3)[:, :, 0].reshape(-1, 64)[rows] * np.repeat(s[:, 0], 16)[rows][:, None] for c, s in ((k, ks), (v, vs)))
        ref, mean, _, _ = R.attention(host(q)[new - 1:new, 0], kk, vv, len(rows) - 1, 0.1, 0)
        assert (np.abs(host(y)[new - 1, 0] - ref[0]) <= 4 * HALF16 * mean[0]).all()


def test_attn_sequence_with_more_rows_than_announced_is_left_out():
    lens = [(30, 1), (40, 3), (50, 1)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(6), lens, 1, 2, 16, 64, torch.float16)
    ws = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 3, 2, 2, 1, 64), dtype=torch.uint8, device=DEV)
    K.attn_q8(q, y, start, kv_len, table, cache, ws, 2, 0.1)
    assert (y[1:4] == 0.5).all() and not (y[0] == 0.5).any() and not (y[4] == 0.5).any()
    assert K.device_error() == 8 and K.device_error() == 0


def test_attn_offsets_beyond_32_bits():
    """A cache of more than 4 GB: the last block is read and written where it stands."""
    blocks, heads, size, dim = 33000, 8, 128, 128
    cache = K.KvCache.empty(blocks, heads, size, dim)
    rng = U.seeded(7)
    x = dev(rng.standard_normal((100, 8, dim)), torch.float16)
    slots = np.arange(100, dtype=np.int32) + (blocks - 1) * size
    K.rope_append_q8(None, x, x, None, dev(slots), cache)
    back = torch.zeros_like(x)
    K.kv_read_q8(cache, dev(slots), back, None)
    assert float((back - x).abs().max()) <= float(x.abs().max()) / 127 + 1e-3
    q = dev(rng.standard_normal((1, 8, dim)), torch.float16)
    y = torch.zeros_like(q)
    ws = torch.empty(K.attn_q8_workspace_bytes(1, 1, 1, 8, 8, dim), dtype=torch.uint8, device=DEV)
    K.attn_q8(q, y, dev(np.array([0, 1], np.int32)), dev(np.array([100], np.int32)), dev(np.array([[blocks - 1]], np.int32)), cache, ws, 1, 0.1)
    kk = host(back)
    for h in range(8):
        ref, mean, _, _ = R.attention(host(q)[:, h], kk[:, h], kk[:, h], 99, 0.1, 0)
        assert (np.abs(host(y)[:, h] - ref) <= 4 * HALF16 * mean).all()
    no_error()


# ------------------------------------------------------------------ sampling

def sample_rows(x, **kw):
    """Runs the rows of x (a device tensor) and compares every token with the reference."""
    n = x.shape[0]
    args = {k: dev(np.asarray(v)).to(torch.int32 if k == "top_k" else torch.float32) for k, v in kw.items() if k != "u"}
    u = dev(np.asarray(kw["u"], np.float32))
    token, logp = torch.full((n,), -9, dtype=torch.int32, device=DEV), torch.zeros(n, device=DEV)
    K.sample(x, u, token, logp, **args)
    xs, token, logp, u = host(x), token.tolist(), host(logp), u.double().cpu().numpy()
    for r in range(n):
        one = {k: (int if k == "top_k" else float)(v[r].item()) for k, v in args.items()}
        t, lp = R.sample(xs[r], u=float(u[r]), **one)
        assert token[r] == t, (r, one, u[r])
        assert (math.isnan(lp) and math.isnan(logp[r])) or abs(logp[r] - lp) <= 2 * HALF32 * (1 + abs(lp)) + 1e-9
    no_error()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (5, 255), (4, 2049), (64, 1000), (1, 32000), (9, 50257), (2, 131072), (400, 4096), (2, 327680)])
def test_sample(f32, rows, vocab):
    rng = U.seeded(rows + vocab)
    x = dev(rng.standard_normal((rows, vocab)) * 3, torch.float32 if f32 else torch.float16)
    u = rng.random(rows).astype(np.float32)
    pick = lambda *v: rng.choice(v, rows)  # noqa: E731
    t = pick(0.0, 0.3, 0.7, 1.0, 2.0)
    sample_rows(x, u=u)
    sample_rows(x, u=u, temperature=t)
    sample_rows(x, u=u, temperature=t, top_k=pick(0, 1, 2, 5, 50, vocab, vocab + 1))
    sample_rows(x, u=u, temperature=t, top_p=pick(0.0, 0.1, 0.5, 0.9, 0.999, 1.0))
    sample_rows(x, u=u, temperature=t, min_p=pick(0.0, 0.01, 0.3, 1.0, 1.5))
    sample_rows(x, u=u, temperature=t, top_k=pick(0, 3, 40), top_p=pick(0.3, 0.95, 1.0), min_p=pick(0.0, 0.02))


@pytest.mark.parametrize("f32", [False, True])
def test_sample_ties_and_ends(f32):
    """Equal logits everywhere, few distinct values, and u at both ends: the lowest index wins every tie."""
    n, vocab = 12, 3001
    rng = U.seeded(8)
    dtype = torch.float32 if f32 else torch.float16
    u = np.array([0.0, 1 - 2.0 ** -24, 0.5, 0.25, 0.999, 1e-7] * 2, np.float32)
    for x in (np.zeros((n, vocab)), rng.integers(-2, 3, (n, vocab)).astype(float), np.where(rng.random((n, vocab)) < 0.5, 0.0, -0.0), np.full((n, vocab), -65504.0)):
        x = dev(x, dtype)
        ones = np.ones(n)
        sample_rows(x, u=u, temperature=0 * ones)
        sample_rows(x, u=u, top_k=np.arange(1, n + 1) * 17)
        sample_rows(x, u=u, top_p=np.linspace(0, 0.99, n))
        sample_rows(x, u=u, top_k=700 * ones, top_p=0.5 * ones)
        sample_rows(x, u=u, top_k=700 * ones, top_p=0.5 * ones, min_p=0.5 * ones)


@pytest.mark.parametrize("f32", [False, True])
def test_sample_masked_and_not_finite(f32):
    vocab = 5000
    rng = U.seeded(9)
    x = rng.standard_normal((9, vocab)) * 2
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 10:] = -np.inf
    x[3, :] = -np.inf
    x[3, 4321] = -3.0
    x[4, ::2] = np.nan
    x[5, [17, 900, 4000]] = np.inf
    x[6] = -65504.0 if not f32 else -3.4028234663852886e38
    x[6, 77] = 1.0
    x[7, :4000] = -np.inf
    x[8] = np.where(rng.random(vocab) < 0.5, -np.inf, 0.0)
    x = dev(x, torch.float32 if f32 else torch.float16)
    u = rng.random(9).astype(np.float32)
    ones = np.ones(9)
    for t in (0.0, 1.0, 1e-30, 50.0):
        sample_rows(x, u=u, temperature=t * ones)
        sample_rows(x, u=u, temperature=t * ones, top_k=20 * ones)
        sample_rows(x, u=u, temperature=t * ones, top_p=0.9 * ones)
        sample_rows(x, u=u, temperature=t * ones, top_k=2000 * ones, top_p=0.9 * ones, min_p=0.01 * ones)


def test_sample_rows_with_strides():
    rng = U.seeded(10)
    wide = dev(rng.standard_normal((6, 1003)), torch.float16)
    for x in (wide[:, :1000], wide[:, 3:], wide[::2, 5:1001]):
        sample_rows(x, u=rng.random(x.shape[0]).astype(np.float32), top_p=np.full(x.shape[0], 0.8))


def test_sample_follows_the_distribution():
    """Evenly spaced u over [0, 1): every token comes up in proportion to its share, within one draw."""
    n, vocab = 4096, 300
    x = dev(np.repeat(U.seeded(11).standard_normal((1, vocab)) * 2, n, 0), torch.float32)
    u = ((torch.arange(n, device=DEV) + 0.5) / n).float()
    token = torch.zeros(n, dtype=torch.int32, device=DEV)
    K.sample(x, u, token)
    share = torch.softmax(x[0].double(), 0) * n
    assert float((torch.bincount(token.long(), minlength=vocab) - share).abs().max()) <= 1.01


# ------------------------------------------------------------------ together

class Served:
    """A small decode loop over the operators: two attention layers of random projections' outputs, paged caches, tokens drawn."""

    def __init__(self, seqs, block, pool, rows, width, heads=2, group=4, dim=64, layers=2, vocab=997):
        i = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
        self.n, self.block, self.heads, self.group, self.dim, self.vocab = seqs, block, heads, group, dim, vocab
        self.ctx, self.new, self.table, self.ring, self.state = i(seqs), i(seqs), i(seqs, width) - 1, torch.arange(pool, dtype=torch.int32, device=DEV), i(2)
        self.state[1] = pool
        self.kv_len, self.start, self.pos, self.slots, self.status = i(seqs), i(seqs + 1), i(rows), i(rows), i(seqs)
        self.caches = [K.KvCache.empty(pool, heads, block, dim) for _ in range(layers)]
        self.x = [torch.zeros(rows, (group + 2) * heads, dim, dtype=torch.float16, device=DEV) for _ in range(layers)]
        self.q = torch.zeros(rows, group * heads, dim, dtype=torch.float16, device=DEV)
        self.y = [torch.zeros_like(self.q) for _ in range(layers)]
        self.rope = K.rope_table(4096, dim, 10000.0)
        self.logits, self.u, self.token = torch.zeros(seqs, vocab, dtype=torch.float16, device=DEV), torch.zeros(seqs, device=DEV), i(seqs)
        self.top_p = torch.full((seqs,), 0.9, device=DEV)
        self.most = rows
        self.ws = torch.empty(K.attn_q8_workspace_bytes(rows, seqs, rows, group * heads, heads, dim), dtype=torch.uint8, device=DEV)

    def step(self):
        K.kv_plan(self.ctx, self.new, self.table, self.ring, self.state, self.state, self.ctx, self.kv_len, self.start, self.pos, self.slots, self.status, self.block)
        for x, cache, y in zip(self.x, self.caches, self.y):
            q, k, v = x.split([self.group * self.heads, self.heads, self.heads], 1)
            K.rope_append_q8(q, k, v, self.q, self.slots, cache, self.rope, self.pos)
            K.attn_q8(self.q, y, self.start, self.kv_len, self.table, cache, self.ws, self.most, 1 / math.sqrt(self.dim))
        K.sample(self.logits, self.u, self.token, None, None, None, self.top_p)


@pytest.mark.parametrize("captured", [False, True])
def test_decode_steps_together(captured):
    """Sequences come, grow, end and give their blocks to others, in one captured graph or step by step; every step's attention
    is compared with a dense one over everything that was appended (within the cache's own rounding)."""
    rng = U.seeded(12)
    s = Served(seqs=5, block=16, pool=24, rows=64, width=8)
    graph = None
    if captured:
        s.step()
        torch.cuda.synchronize()
        s.ctx.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.step()
    held = [[[], []] for _ in range(5)]          # per sequence and layer: the rows of (rotated k, v) appended
    for step in range(14):
        new = np.array([1 if len(h[0]) else 0 for h in held])
        for b in range(5):
            if not new[b] and rng.random() < 0.5:
                new[b] = rng.integers(1, 12)     # a prompt
            elif len(held[b][0]) > 40:
                new[b] = -1
        s.new.copy_(dev(new.astype(np.int32)))
        for x in s.x:
            x.copy_(dev(rng.standard_normal(x.shape)))
        s.logits.copy_(dev(rng.standard_normal(s.logits.shape) * 2))
        s.u.copy_(dev(rng.random(5).astype(np.float32)))
        graph.replay() if captured else s.step()
        torch.cuda.synchronize()
        assert not s.status.any()
        start, table = s.start.tolist(), host(s.rope)
        for layer, (x, y) in enumerate(zip(s.x, s.y)):
            x, y = host(x), host(y)
            for b in range(5):
                rows = slice(start[b], start[b + 1])
                if new[b] == -1:
                    held[b][layer] = []
                    continue
                n0 = len(held[b][layer])
                pos = n0 + np.arange(max(new[b], 0))
                assert start[b + 1] - start[b] == len(pos) and s.pos[rows].tolist() == pos.tolist()
                turned = R.rope(x[rows, :10], table, pos, False)
                held[b][layer] += [(turned[i, 8:10], x[rows, 10:][i]) for i in range(len(pos))]
                if not len(pos):
                    continue
                k, v = (np.stack([r[j] for r in held[b][layer]]) for j in (0, 1))
                for g in range(8):
                    kk, vv = k[:, g // 4], v[:, g // 4]
                    ref, mean, _, _ = R.attention(turned[:, g].astype(np.float16).astype(np.float64), kk, vv, n0, 0.125, 0)
                    # a code is off by at most one step 2 max / 127 (its own half step and a grown scale's): the keys' part
                    # moves a score by sum |q| of that, twice that a weight, and the values' part adds itself
                    key_step, val_step = 2 * np.abs(kk).max() / 127, 2 * np.abs(vv).max() / 127
                    tol = (np.exp(2 * 0.125 * key_step * np.abs(turned[:, g]).sum(1)) - 1)[:, None] * 2 * mean + val_step + 4 * HALF16 * mean
                    assert (np.abs(y[rows][:, g] - ref) <= tol).all()
        assert s.token.tolist() == [R.sample(host(s.logits)[b], top_p=float(s.top_p[b]), u=float(s.u[b]))[0] for b in range(5)]
        # no block belongs to two
        used = [t for b in range(5) for t in s.table[b, :-(-int(s.ctx[b]) // 16)].tolist()]
        free = [int(s.ring[(int(s.state[0]) + i) % 24]) for i in range(int(s.state[1]))]
        assert sorted(used + free) == list(range(24))
    no_error()


def test_projection_stack_with_attention():
    """Decode steps of an 8B-shaped layer, captured once: O reads the attention over what the QKV projection wrote in every
    step; a sequence that ends gives its blocks back and begins anew."""
    from ztensor_b200.stack import DecodeAttention, ProjectionStack
    st = ProjectionStack("llama3-8b", batch=2, layers=1)
    att = DecodeAttention(st, blocks=5, block_size=16, max_positions=64)
    st.step(attention=att)                       # loads the kernels
    att.ctx.zero_(), att.ring_state.copy_(torch.tensor([0, 5], device=DEV))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st.step(attention=att)
    torch.cuda.synchronize()
    att.ctx.zero_(), att.ring_state.copy_(torch.tensor([0, 5], device=DEV))
    rng, held, table = U.seeded(15), [[], []], host(att.rope)
    for step in range(40):
        att.new.copy_(torch.tensor([1, -1 if step == 20 else 1], device=DEV))
        st.x["qkv"].copy_(dev(rng.standard_normal((2, 4096))))
        before = st.x["o"].clone()
        graph.replay()
        torch.cuda.synchronize()
        assert att.status.tolist() == [0, 0] and att.positions.tolist()[0] == len(held[0])
        if step == 20:
            held[1] = []
            assert torch.equal(st.x["o"][1], before[1])
        # the queries were rotated in place; keys and values stand in y as the projection left them
        y, out = host(st.y["qkv"]).reshape(2, 48, 128), host(st.x["o"]).reshape(2, 32, 128)
        for b in range(1 if step == 20 else 2):
            held[b].append((R.rope(y[b:b + 1, 32:40], table, np.array([len(held[b])]), False)[0], y[b, 40:]))
            k, v = (np.stack([r[j] for r in held[b]]) for j in (0, 1))
            for h in range(0, 32, 5):
                kk, vv = k[:, h // 4], v[:, h // 4]
                ref, mean, _, _ = R.attention(y[b:b + 1, h], kk, vv, len(kk) - 1, 128 ** -0.5, 0)
                key_step, val_step = 2 * np.abs(kk).max() / 127, 2 * np.abs(vv).max() / 127       # as in the loop of decode steps above
                tol = (np.exp(2 * 128 ** -0.5 * key_step * np.abs(y[b, h]).sum()) - 1) * 2 * mean + val_step + 4 * HALF16 * mean
                assert (np.abs(out[b, h] - ref[0]) <= tol[0]).all()
    no_error()


def test_calls_without_rows_do_nothing():
    cache = random_cache(U.seeded(14), 4, 2, 16, 64)
    before = [t.clone() for t in cache.tensors]
    i = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
    h = lambda heads: torch.zeros(0, heads, 64, dtype=torch.float16, device=DEV)  # noqa: E731
    table = K.rope_table(4, 64, 10000.0)
    K.rope(h(3), h(3), table, i(0))
    K.rope_append_q8(h(8), h(2), h(2), h(8), i(0), cache, table, i(0))
    K.kv_read_q8(cache, i(0), h(2), h(2))
    K.attn_q8(h(8), h(8), i(3), i(2), i(2, 1), cache, torch.empty(K.attn_q8_workspace_bytes(0, 2, 1, 8, 2, 64), dtype=torch.uint8, device=DEV), 1, 0.1)
    K.sample(torch.zeros(0, 9, device=DEV), torch.zeros(0, device=DEV), i(0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, cache.tensors))
    no_error()


def test_two_streams_at_once():
    """Two attention calls on two streams with a workspace each give what each gives alone."""
    cases = [attn_run([(3000, 1), (77, 1)], 2, 8, 16, 128, seed=20 + i) for i in range(2)]
    want = [c[0][5].clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, ws), st in zip(cases, streams):
            with torch.cuda.stream(st):
                K.attn_q8(c[4], c[5], c[2], c[3], c[1], c[0], ws, 1, 1 / math.sqrt(128))
    torch.cuda.synchronize()
    assert all(torch.equal(c[0][5], w) for c, w in zip(cases, want))
    no_error()


def test_same_inputs_same_bits():
    case, ws = attn_run([(5000, 1), (777, 1), (4096, 1)], 4, 8, 64, 128, seed=30)
    cache, table, start, kv_len, q, y = case
    want = y.clone()
    for _ in range(5):
        y.fill_(9)
        K.attn_q8(q, y, start, kv_len, table, cache, ws, 1, 1 / math.sqrt(128))
        assert torch.equal(y[:3], want[:3])


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.rope(x, x, torch.zeros(4, 32, 2, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="current CUDA device"):
        K.sample(torch.zeros(1, 9), torch.zeros(1, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    assert _lib.lib().ztq_check_sm100() == 1
