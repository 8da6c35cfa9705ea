"""Attention and the operators around it at values far from one: queries and scales of any size, blocks that a row does not see, refused sequences."""
import math

import numpy as np
import pytest
import torch

from tests import step_ref as R
from tests import util as U
from tests.test_gpu_step import DEV, FEW, HALF16, HALF32, MANY, MIXED, ONE, attn_case, dev, host, no_error
from ztensor_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def a_clean_error_word():
    K.device_error()


def run(lens, cache, table, start, kv_len, q, y, scale, window=0, most=None):
    most = most or max(1, max(a for _, a in lens))
    ws = torch.full((K.attn_q8_workspace_bytes(q.shape[0], len(lens), most, q.shape[1], cache.kv_heads, cache.head_dim) // 4,), math.nan, device=DEV)
    K.attn_q8(q, y, start, kv_len, table, cache, ws, most, scale, window)


def check(lens, cache, table, q, y, scale, window=0, f32=False, rows=None):
    """Every row against 64 bits.  The bound holds for values of any size, because each part of it is relative to what the row itself sees:
      a score is an fp32 sum of D / 16 + 2 roundings, its query is held to 2^-22 of itself (fp32: two fp16 terms) or exactly, and an element far
          below the row's largest to 2^-39 of that one (fp16's last step below 2^15);
      a weight has fp16's half step, or that of two terms, and a few roundings of the exponential;
      a weight times its V scale far below the row's largest such product ends at fp16's last half step, 2^-25, where the largest is held as 2^4
          (fp32: 2^12) within a factor of 2^0.5;
      sums over n keys take n / 16 more roundings of 2^-23; the output has its own half step."""
    codes_k, codes_v, ks, vs = (host(t).astype(np.float64) for t in cache.tensors)
    size, dim, group = cache.block_size, cache.head_dim, q.shape[1] // cache.kv_heads
    got, qh, table = host(y), host(q), table.cpu().numpy()
    row = 0
    for b, (n, a) in enumerate(lens):
        block, at = table[b][np.arange(n) // size], np.arange(n) % size
        there = (block >= 0) & (block < cache.blocks)
        block = np.where(there, block, 0)
        for h in range(cache.kv_heads):
            kk, cv, sv = codes_k[block, h, at] * ks[block, h][:, None], codes_v[block, h, at], vs[block, h]
            for i in range(a):
                if rows is not None and i not in rows:
                    continue
                pos = n - a + i
                seen = there & (np.arange(n) <= pos) & (np.arange(n) > pos - window if window else True)
                for g in range(h * group, (h + 1) * group):
                    out = got[row + i, g]
                    if not seen.any():
                        assert (out == 0).all()
                        continue
                    x = qh[row + i, g]
                    s = kk[seen] @ x * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    w, c = p * sv[seen], cv[seen]
                    ref, mean = w @ c, np.abs(w) @ np.abs(c)
                    reach = abs(scale) * (np.abs(kk[seen]) @ np.abs(x)).max()
                    far = abs(scale) * np.abs(kk[seen]).sum(1).max() * np.abs(x).max() * 2.0 ** -39 if f32 else 0.0
                    score = (dim / 16 + 2) * 2 * HALF32 * reach + (2.0 ** -22 * reach if f32 else 0.0) + far
                    weight = score + (4 * 2.0 ** -22 if f32 else HALF16) + (64 + seen.sum() / 8) * HALF32
                    ends = 2.0 ** (-36.5 if f32 else -28.5) * np.abs(w).max() * np.abs(c).sum(0)
                    tol = 2 * weight * mean + ends + (2.0 ** -126 if y.dtype is torch.float32 else HALF16 * np.abs(ref) + 2.0 ** -25)
                    worst = np.abs(out - ref) / tol
                    if y.dtype is torch.float16:     # from 65520 on, half a step above its largest number, fp16 rounds to infinity
                        worst = np.where(np.abs(ref) + tol < 65520, worst, np.where(np.isinf(out), out * ref < 0, (np.abs(ref) - tol >= 65520) + worst))
                    assert (worst <= 1).all(), (b, i, g, float(np.nanmax(worst)), out[:4], ref[:4])
        row += a
    assert (got[row:] == 0.5).all()


# ------------------------------------------------------------------ fp32 queries of any size

ROWS = [(200, 1), (77, 1), (33, 1)]                  # few rows per kv head
PROMPT = [(300, 40), (90, 64)]


@pytest.mark.parametrize("dim,lens", [(64, ROWS), (128, ROWS), (256, ROWS), (64, FEW), (256, PROMPT), (64, PROMPT), (128, PROMPT)])
@pytest.mark.parametrize("size", [1e-30, 3e-8, 1e-5, 1e-3, 6e4, 1e6, 1e30])
def test_fp32_queries_of_any_size(dim, lens, size):
    """The keys' scales are as far the other way, so that the scores stay of order one."""
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32)
    q *= size
    cache.tensors[2].mul_(2.0 ** -round(math.log2(size)))
    run(lens, cache, table, start, kv_len, q, y, 1 / math.sqrt(dim))
    check(lens, cache, table, q, y, 1 / math.sqrt(dim), f32=True)
    no_error()


@pytest.mark.parametrize("dim,lens", [(64, ROWS), (128, FEW), (256, FEW), (64, PROMPT), (128, PROMPT)])
def test_fp32_rows_and_elements_of_different_sizes(dim, lens):
    """Each row has a size of its own, and some have one element far above the others; rows of zeros and of subnormal numbers among them."""
    rng = U.seeded(dim + 1)
    cache, table, start, kv_len, q, y = attn_case(rng, lens, 2, 4, 32, dim, torch.float32)
    x = host(q) * np.exp2(rng.integers(-40, 3, q.shape[:2]))[..., None]
    x[::3, 1, dim // 3] *= 2.0 ** 20
    x[::4, 2] = 0
    x[::2, 3] *= 2.0 ** -110
    q.copy_(dev(x))
    run(lens, cache, table, start, kv_len, q, y, 0.1)
    check(lens, cache, table, q, y, 0.1, f32=True)
    no_error()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [ROWS, PROMPT], ids=["rows", "prompt"])
def test_fp32_queries_that_are_not_finite(dim, lens):
    """Such a row is NaN; the others are as without it."""
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32)
    q[1, 3, 5], q[0, 6, 1] = math.inf, math.nan
    run(lens, cache, table, start, kv_len, q, y, 0.1)
    assert torch.isnan(y[1, 3]).all() and torch.isnan(y[0, 6]).all() and not torch.isnan(y[2:]).any()
    got = y.clone()
    q[1, 3, 5], q[0, 6, 1] = 0.0, 0.0
    y.fill_(0.5)
    run(lens, cache, table, start, kv_len, q, y, 0.1)
    check(lens, cache, table, q, y, 0.1, f32=True)
    got[1, 3], got[0, 6] = y[1, 3], y[0, 6]
    assert torch.equal(got, y)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("x32,y32", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("lens,window", [([(3000, 260)], 0), ([(5000, 150), (3, 2), (2100, 90)], 0), ([(4100, 33)], 2500)])
def test_fp32_prompts_with_their_keys_in_ranges(dim, x32, y32, lens, window):
    cache, table, start, kv_len, q, y = attn_case(U.seeded(7), lens, 1, 4, 64, dim, torch.float32 if x32 else torch.float16)
    y = torch.full(q.shape, 0.5, dtype=torch.float32 if y32 else torch.float16, device=DEV)
    run(lens, cache, table, start, kv_len, q, y, 0.05, window)
    check(lens, cache, table, q, y, 0.05, window, f32=True, rows=range(0, 300, 13))
    no_error()


@pytest.mark.parametrize("heads,group,dim", [(4, 4, 64), (4, 3, 128), (4, 2, 256)])
def test_fp32_batches_that_two_kernels_share(heads, group, dim):
    cache, table, start, kv_len, q, y = attn_case(U.seeded(9), MIXED, heads, group, 64, dim, torch.float32)
    run(MIXED, cache, table, start, kv_len, q, y, 1 / math.sqrt(dim))
    check(MIXED, cache, table, q, y, 1 / math.sqrt(dim), f32=True, rows=range(0, 80, 17))
    no_error()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 50])
def test_fp32_scales_of_any_kind(new, dim):
    lens = [(300, new), (50 + new, new)]
    rng = U.seeded(13)
    cache, table, start, kv_len, q, y = attn_case(rng, lens, 2, 4, 16, dim, torch.float32)
    for t in cache.tensors[2:]:
        t.copy_(dev((rng.uniform(0.5, 1.5, t.shape) * np.exp2(rng.integers(-16, -4, t.shape)) * rng.choice([1, 1, 1, -1, 0], t.shape)).astype(np.float32)))
    for scale in (0.1, -0.1, 0.0):
        run(lens, cache, table, start, kv_len, q, y, scale)
        check(lens, cache, table, q, y, scale, f32=True)
    no_error()


# ------------------------------------------------------------------ V scales far apart

@pytest.mark.parametrize("f32,small", [(False, -16), (True, -16), (True, -60)])
@pytest.mark.parametrize("dim,new", [(64, 1), (64, 40), (128, 40), (128, 3), (256, 20)])
@pytest.mark.parametrize("where", [0, 1, 2])
def test_steps_without_v_scales(f32, small, dim, new, where):
    """All V scales of 128 tokens are zero, in front of, between or behind tokens of small ones."""
    lens = [(128 * 3, new)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32 if f32 else torch.float16)
    cache.tensors[3].mul_(2.0 ** (small + 7))
    cache.tensors[3][table[0, 8 * where:8 * where + 8].long()] = 0.0
    run(lens, cache, table, start, kv_len, q, y, 0.05)
    check(lens, cache, table, q, y, 0.05, f32=f32)
    no_error()


@pytest.mark.parametrize("f32,small", [(False, -16), (True, -60)])
@pytest.mark.parametrize("dim,new", [(64, 1), (64, 40), (128, 40)])
def test_steps_without_blocks(f32, small, dim, new):
    lens = [(128 * 3, new)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32 if f32 else torch.float16)
    cache.tensors[3].mul_(2.0 ** (small + 7))
    table[0, 8:16] = -1
    run(lens, cache, table, start, kv_len, q, y, 0.05)
    check(lens, cache, table, q, y, 0.05, f32=f32)
    assert K.device_error() == 7


@pytest.mark.parametrize("huge", [2.0 ** 40, 1e20, 3e38])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dim,new", [(64, 1), (64, 9), (64, 40), (128, 5), (128, 40), (256, 3)])
def test_huge_scales_in_front_of_the_window(huge, f32, dim, new):
    """Blocks that slid out of the window are in the table still."""
    lens, window = [(300, new), (140, new)], 60
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32 if f32 else torch.float16)
    for b, (n, _) in enumerate(lens):
        gone = table[b, :(n - new - window + 1) // 16].long()
        cache.tensors[2][gone] = huge
        cache.tensors[3][gone] = -huge
    run(lens, cache, table, start, kv_len, q, y, 0.05, window)
    check(lens, cache, table, q, y, 0.05, window, f32=f32)
    no_error()


@pytest.mark.parametrize("huge", [2.0 ** 24, 1e20, 2e36])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dim,new", [(64, 20), (64, 5), (64, 70), (128, 18), (128, 70), (256, 18)])
@pytest.mark.parametrize("window", [0, 30])
def test_huge_scales_that_only_some_rows_see(huge, f32, dim, new, window):
    """The last block's values are far above all others: the rows in front of it do not see them, and with a window the last rows do not see
    a block in front that the first ones do."""
    n = 96 + new
    lens = [(n, new)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32)
    if not f32:
        q, y = q.half(), y.half()
    cache.tensors[3][table[0, (n - 1) // 16].long()] *= huge
    if window:
        cache.tensors[3][table[0, (n - new - 3) // 16].long()] *= huge
    y = y.float()                                # the large ones leave fp16's range
    run(lens, cache, table, start, kv_len, q, y, 0.05, window)
    check(lens, cache, table, q, y, 0.05, window, f32=True)
    no_error()


@pytest.mark.parametrize("dim,new", [(64, 18), (64, 70), (128, 18), (128, 70), (256, 18)])
def test_fp16_rows_that_do_not_see_the_large_scales(dim, new):
    n = 96 + new
    lens = [(n, new)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float16)
    cache.tensors[3].mul_(2.0 ** -6)
    last = (n - 1) // 16
    cache.tensors[3][table[0, last].long()] *= 2.0 ** 12
    run(lens, cache, table, start, kv_len, q, y, 0.05)
    check(lens, cache, table, q, y, 0.05)
    no_error()


@pytest.mark.parametrize("power,apart", [(36, (44, 20, -40)), (12, (44, 20, -40)), (12, (80, 60, -75)), (12, (-60, 10, -60))])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dim,new", [(64, 1), (64, 20), (128, 5), (128, 70), (256, 2)])
def test_a_huge_scale_under_a_vanishing_weight(power, apart, f32, dim, new):
    """One block's keys point away from the queries, so its weights vanish beside the others', and its V scale makes up for a part of that."""
    lens = [(200, new)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, 16, dim, torch.float32 if f32 else torch.float16)
    q.copy_(q.abs() + 0.25)
    cache.tensors[3].mul_(2.0 ** power)
    for j, more, sign in zip((4, 9, 10), apart, (-1, -1, 1)):
        block = int(table[0, j])
        cache.tensors[0][block].clamp_(20, 127)
        cache.tensors[0][block].mul_(sign)
        cache.tensors[2][block] = 2.0 ** -6
        cache.tensors[3][block] *= 2.0 ** more
    scale = 60 / (dim * 1.5 * 2.0 ** -6 * 70)    # scores of the blocks around -60 and 60
    run(lens, cache, table, start, kv_len, q, y, scale)
    check(lens, cache, table, q, y, scale, f32=f32)
    no_error()


# ------------------------------------------------------------------ what a window has left behind

@pytest.mark.parametrize("dim,size", [(64, 16), (128, 64), (256, 32), (64, 128)])
@pytest.mark.parametrize("new", [1, 5, 40, 90])
@pytest.mark.parametrize("window", [1, 17, 100])
def test_blocks_in_front_of_the_window_may_be_gone(dim, size, new, window):
    """A server gives back the blocks in front of the window and marks them -1: nobody sees them, so there is no error."""
    lens = [(700, new), (90 + new, new), (1, 1)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(dim), lens, 2, 4, size, dim, torch.float16)
    for b, (n, a) in enumerate(lens):
        table[b, :max(0, n - a - window + 1) // size] = -1
    run(lens, cache, table, start, kv_len, q, y, 0.1, window)
    check(lens, cache, table, q, y, 0.1, window)
    no_error()


# ------------------------------------------------------------------ behind one another

@pytest.mark.parametrize("captured", [False, True])
def test_prompt_attention_between_tensor_core_products(captured):
    """Kernels that hold all of an SM's tensor memory, started in one another's shadow: attention over a prompt between products."""
    from oracle import oracle as O
    from tests import gpu_util as G
    lens, n, k = [(600, 300)], 512, 1024
    cache, table, start, kv_len, q, y = attn_case(U.seeded(3), lens, 8, 4, 64, 128, torch.float16)
    rng = U.seeded(4)
    qd, meta = G.upload_w4g(O.quantize_gptq(U.make_weights(rng, n, k), 128))
    x, out = torch.randn(32, k, device=DEV).half(), torch.zeros(32, n, device=DEV)
    ws, want = torch.empty(K.gemm_w4g_tc_workspace_bytes(n, k, 32), dtype=torch.uint8, device=DEV), torch.zeros(32, n, device=DEV)
    work = torch.empty(K.attn_q8_workspace_bytes(q.shape[0], 1, 300, 32, 8, 128), dtype=torch.uint8, device=DEV)
    K.gemm_w4g_tc(qd, meta, x, want, n, k, 128, 32, ws, K.Y_F32)
    K.attn_q8(q, y, start, kv_len, table, cache, work, 300, 0.1)
    first = y.clone()
    check(lens, cache, table, q, y, 0.1, rows=range(0, 300, 41))

    def step():
        for _ in range(3):
            K.gemm_w4g_tc(qd, meta, x, out, n, k, 128, 32, ws, K.Y_F32)
            K.attn_q8(q, y, start, kv_len, table, cache, work, 300, 0.1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph):
            step()
    for _ in range(20):
        y.fill_(0.5), out.zero_()
        graph.replay() if captured else step()
    torch.cuda.synchronize()
    assert torch.equal(y, first) and torch.equal(out, want)
    no_error()


# ------------------------------------------------------------------ the ends of a sequence

@pytest.mark.parametrize("positions", [50, 64])
def test_decode_attention_up_to_its_last_position(positions):
    """A table rounded up to whole blocks takes more positions than were asked for; all that it takes are right."""
    from ztensor_b200.stack import DecodeAttention, ProjectionStack
    st = ProjectionStack("llama3-8b", batch=1, layers=1)
    att = DecodeAttention(st, blocks=5, block_size=16, max_positions=positions)
    assert att.table.shape[1] == 4
    rng, held, rope = U.seeded(15), [], host(K.rope_table(64, 128, 500000.0))
    for step in range(64):
        st.x["qkv"].copy_(dev(rng.standard_normal((1, 4096))))
        st.step(attention=att)
        torch.cuda.synchronize()
        assert att.status.tolist() == [0] and att.positions.tolist() == [step]
        z, out = host(st.y["qkv"]).reshape(1, 48, 128), host(st.x["o"]).reshape(32, 128)
        held.append((R.rope(z[:, 32:40], rope, np.array([step]), False)[0], z[0, 40:]))
        k, v = (np.stack([r[j] for r in held]) for j in (0, 1))
        for h in range(0, 32, 5):
            kk, vv = k[:, h // 4], v[:, h // 4]
            ref, mean, _, _ = R.attention(z[:, h], kk, vv, step, 128 ** -0.5, 0)
            # a code is off by at most one step, 2 max / 127: the keys' moves a score, the values' adds itself
            key_step, val_step = 2 * np.abs(kk).max() / 127, 2 * np.abs(vv).max() / 127
            tol = (np.exp(2 * 128 ** -0.5 * key_step * np.abs(z[0, h]).sum()) - 1) * 2 * mean + val_step + 4 * HALF16 * mean
            assert (np.abs(out[h] - ref[0]) <= tol[0]).all(), (step, h)
    no_error()


@pytest.mark.parametrize("x32", [False, True])
def test_refused_sequences_raise_no_error(x32):
    """A sequence whose table is full gets status 2 and no slots: its rows' positions lie behind the rotary table, which is no error; a row with a
    slot there is one."""
    dtype = torch.float32 if x32 else torch.float16
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    z = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    kv_len, start, pos, slots, status, nxt = z(3), z(4), z(40), z(40), z(3), z(3)
    table = i(0, 1, 2, 3, -1, -1).view(3, 2)
    K.kv_plan(i(32, 20, 0), i(1, 5, 34), table, i(4, 5, 0, 1, 2, 3), i(0, 2), z(2), nxt, kv_len, start, pos, slots, status, 16)
    assert status.tolist() == [2, 0, 2] and pos.tolist()[:7] == [32, 20, 21, 22, 23, 24, 0] and slots.tolist()[:2] == [-1, 52]
    cache, rope = K.KvCache.empty(6, 1, 16, 64), K.rope_table(32, 64, 10000.0)
    x = torch.randn(40, 4, 64, device=DEV).to(dtype)
    q, k, v = x.split([2, 1, 1], 1)
    out = torch.zeros(40, 2, 64, dtype=dtype, device=DEV)
    K.rope_append_q8(q, k, v, out, slots, cache, rope, pos)
    no_error()
    assert torch.isfinite(out[1:38]).all()
    y = torch.full_like(out, 0.5)
    K.attn_q8(out, y, start, kv_len, table, cache, torch.empty(K.attn_q8_workspace_bytes(40, 3, 40, 2, 1, 64), dtype=torch.uint8, device=DEV), 40, 0.125)
    assert (y[0] == 0).all() and torch.isfinite(y).all() and (y[6:] == 0).all()
    no_error()
    slots[0] = 5 * 16
    K.rope_append_q8(q, k, v, out, slots, cache, rope, pos)
    assert K.device_error() == 6 and K.device_error() == 0 and torch.isnan(out[0]).all()


def test_device_error_clears_everything():
    """Errors of several operators before one look at the error word: it names one of them, and nothing is left behind."""
    rope = K.rope_table(10, 64, 10000.0)
    x = torch.ones(1, 2, 64, device=DEV)
    K.rope(x, torch.zeros_like(x), rope, torch.tensor([10], dtype=torch.int32, device=DEV))
    lens = [(40, 1)]
    cache, table, start, kv_len, q, y = attn_case(U.seeded(5), lens, 1, 2, 16, 64, torch.float16)
    table[0, 1] = -5
    run(lens, cache, table, start, kv_len, q, y, 0.1)
    assert K.device_error() in (6, 7) and K.device_error() == 0


# ------------------------------------------------------------------ scales that are not finite, in fp32

@pytest.mark.parametrize("dim,new", [(64, 3), (64, 40), (128, 3), (128, 40), (256, 3)])
@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_fp32_scales_that_are_not_finite(dim, new, which, bad):
    """Blocks in front of the window and unused ones change nothing; the last block makes the rows that see it NaN, and no others."""
    n, window = 64 + new, 40
    cache, table, start, kv_len, q, y = attn_case(U.seeded(4), [(n, new)], 2, 4, 16, dim, torch.float32)
    gone = [b for b in range(cache.blocks) if b not in table[0].tolist()] + table[0, :(n - new - window + 1) // 16].tolist()
    for t in cache.tensors[2:]:
        t[gone] = bad
    run([(n, new)], cache, table, start, kv_len, q, y, 0.1, window)
    for t in cache.tensors[2:]:
        t[gone] = 1.0
    check([(n, new)], cache, table, q, y, 0.1, window, f32=True)
    cache.tensors[which][int(table[0, (n - 1) // 16]), 1] = bad
    y.fill_(0.5)
    run([(n, new)], cache, table, start, kv_len, q, y, 0.1, window)
    nan = torch.isnan(y[:new])
    sees = torch.arange(64, n, device=DEV) >= (n - 1) // 16 * 16
    assert not nan[:, :4].any() and torch.equal(nan[:, 4:].any(-1), sees[:, None].expand(-1, 4))
    assert which == 2 or torch.equal(nan[:, 4:].all(-1), sees[:, None].expand(-1, 4))
    no_error()


# ------------------------------------------------------------------ sampling

@pytest.mark.parametrize("f32", [False, True])
def test_tokens_too_light_to_count(f32):
    """A weight below 2^-45 of the largest is 0 and is not drawn, the smallest above that is: at uniform 0 the first token that has any."""
    x = torch.full((4, 300), -40.0, dtype=torch.float32 if f32 else torch.float16, device=DEV)
    x[:, 200] = 0.0
    x[1, 100], x[2, 100], x[3, 7] = -31.0, -30.0, -60.0      # log2: 44.7, 43.3, 86.6
    token = torch.zeros(4, dtype=torch.int32, device=DEV)
    K.sample(x, torch.zeros(4, device=DEV), token)
    assert token.tolist() == [200, 100, 100, 200]
    no_error()
