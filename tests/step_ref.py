"""Plain 64-bit references of the decode-step operators (numpy, one sequence and one row at a time)."""
from __future__ import annotations

import math

import numpy as np


def kv_plan(ctx, new, table, ring, state, block, rows):
    """-> dict of everything ztq_kv_plan writes; `table` and `ring` are not changed."""
    n, width, pool = len(ctx), table.shape[1], len(ring)
    table, out_ring = table.copy(), ring.copy()
    head, count = int(state[0]) % pool, min(max(int(state[1]), 0), pool)
    start, status, kv, nxt = [0], [], [], []
    asked = taken = released = end = 0
    positions, slots = np.zeros(rows, np.int32), np.full(rows, -1, np.int32)
    up = lambda a: -(-a // block)  # noqa: E731
    for b in range(n):
        c, a = int(ctx[b]), int(new[b])
        bad = c < 0 or a < -1 or up(c) > width
        gone = not bad and a == -1
        a = 0 if bad or a < 0 else a
        first, end = end, end + a
        st, ask = 4 if bad else 0, 0
        if a > 0:
            st = 3 if end > rows else 2 if up(c + a) > width else 0
            if st == 0:
                ask = up(c + a) - up(c)
                if ask and asked + ask > count:
                    st = 1
        if ask and st == 0:
            for k in range(ask):
                table[b, up(c) + k] = ring[(head + asked + k) % pool]
            taken = asked + ask
        asked += ask
        if gone:
            for k in range(up(c)):
                if released + k < pool - count:
                    out_ring[(head + count + released + k) % pool] = table[b, k]
            released += up(c)
        for i in range(a):
            if first + i < rows:
                positions[first + i] = c + i
                if st == 0:
                    blk = int(table[b, (c + i) // block])
                    if 0 <= blk < pool:
                        slots[first + i] = blk * block + (c + i) % block
        start.append(min(end, rows))
        status.append(st)
        kv.append(c + a if st == 0 and not gone else 0)
        nxt.append(0 if gone else c + a if st == 0 else c)
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return dict(block_table=table, ring=out_ring, ring_state_out=i32([(head + taken) % pool, count - taken + min(released, pool - count)]), query_start=i32(start),
                status=i32(status), kv_len=i32(kv), next_len=i32(nxt), positions=positions, slots=slots)


def frequencies(rot, base, scaling="none", factor=1.0, low=1.0, high=4.0, original=0.0):
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "by_turns":
        keep = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f * keep + f / factor * (1 - keep)
    if scaling == "by_dim":
        at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        a, b = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
        s = np.clip((i - a) / max(b - a, 0.001), 0, 1)
        return f * (1 - s) + f / factor * s
    return f


def rope(x, table, positions, pairs):
    """x [tokens, heads, dim] float64, table [rows, rot/2, 2]."""
    y = x.astype(np.float64).copy()
    n = table.shape[1]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if pairs else (slice(0, n), slice(n, 2 * n))
    cos, sin = (table[positions, :, i].astype(np.float64)[:, None] for i in (0, 1))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    return y


def scale_for(amax):
    if not np.isfinite(amax):
        return math.nan
    return 2.0 ** -126 if amax == 0 else max(2.0 ** math.ceil(math.log2(amax / 127)), 2.0 ** -126)


def append(codes, scale, x, slots):
    """codes [blocks, heads, size, dim] int8 and scale [blocks, heads] float32 after rows x [tokens, heads, dim] at slots."""
    codes, scale = codes.copy(), scale.astype(np.float64).copy()
    size = codes.shape[2]
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] // size == slots[t] // size:
            n += 1
        b, off = slots[t] // size, slots[t] % size
        for h in range(codes.shape[1]):
            rows = x[t:t + n, h]
            need = scale_for(np.abs(rows).max() if np.isfinite(rows).all() else math.inf)
            had = scale[b, h]
            s = need if off == 0 or math.isnan(need) else had if math.isnan(had) else max(had, need)
            if math.isnan(s):
                codes[b, h, off:off + n] = 0
            else:
                if off and s != had:
                    codes[b, h, :off] = np.rint(codes[b, h, :off] * (had / s))
                codes[b, h, off:off + n] = np.clip(np.rint(rows / s), -127, 127)
            scale[b, h] = s
        t += n
    return codes, scale.astype(np.float32)


def attention(q, k, v, first, scale, window):
    """q [rows, dim] at positions first, first + 1, ..; k, v [keys, dim] -> (y, sum p |v| / sum p, largest scale * sum |q k|, sum |v|)."""
    y, a, t, z = np.zeros_like(q), np.zeros_like(q), 0.0, np.zeros_like(q)
    for i in range(len(q)):
        hi = min(first + i + 1, len(k))
        lo = max(0, first + i - window + 1) if window else 0
        if hi <= lo:
            continue
        s = k[lo:hi] @ q[i] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        y[i], a[i], z[i] = p @ v[lo:hi], p @ np.abs(v[lo:hi]), np.abs(v[lo:hi]).sum(0)
        t = max(t, float((np.abs(k[lo:hi]) @ np.abs(q[i])).max() * abs(scale)))
    return y, a, t, z


def sample(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """x [vocab] float64 -> (token, logprob)."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, math.nan
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return int(order[0]), 0.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = (x[order] == np.inf).astype(np.float64) if top == np.inf else np.where(x[order] == -np.inf, 0.0, np.exp((x[order] - top) / temperature))
    if top_p < 1:
        n = max(1, int((np.concatenate([[0.0], np.cumsum(w)[:-1]]) < top_p * w.sum()).sum()))
        order, w = order[:n], w[:n]
    if min_p > 0:
        keep = w >= min(min_p, 1.0)
        order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    upto = np.cumsum(w)
    i = int(np.searchsorted(upto, min(max(u, 0.0), 1 - 2.0 ** -24) * upto[-1], side="right"))
    return int(order[i]), math.log(w[i] / upto[-1])
