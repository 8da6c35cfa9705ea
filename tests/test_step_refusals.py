"""Arguments that the decode-step entry points refuse, before any device is touched: every case changes one argument of a call
that is otherwise accepted."""
import ctypes as C

import pytest
import torch

from ztensor_b200 import _lib
from ztensor_b200 import kernels as K

INVALID = 1                      # cudaErrorInvalidValue
P = 1 << 20                      # an aligned address nobody reads: refused calls end before it is used


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, block_stride=8 * 16 * 128, blocks=10, kv_heads=8, block_size=16, head_dim=128) | kw
    return K.ZtqKvCache(*[d[n] for n, _ in K.ZtqKvCache._fields_])


def spec(**kw):
    d = dict(base=1e4, factor=2.0, turns_low=1.0, turns_high=4.0, original_positions=4096.0, magnitude=0.0, rot_dim=64, scaling=2) | kw
    return K.ZtqRopeSpec(*[d[n] for n, _ in K.ZtqRopeSpec._fields_])


CALLS = {
    "ztq_kv_plan": dict(ctx_len=P, new_len=P, block_table=P, ring=P, ring_state=P, ring_state_out=P, next_len=P, kv_len=P, query_start=P, positions=P, slots=P, status=P,
                        sequences=4, table_width=8, block_size=16, pool_blocks=64, max_tokens=32, flags=0, stream=None),
    "ztq_rope_table": dict(table=P, first=0, rows=10, spec=spec(), flags=0, stream=None),
    "ztq_rope": dict(x=P, y=2 * P, tokens=4, heads=8, head_dim=128, x_token=1024, x_head=128, y_token=1024, y_head=128, table=P, table_rows=100, rot_dim=128, positions=P, flags=0, stream=None),
    "ztq_rope_append_q8": dict(q=P, k=P, v=P, q_out=2 * P, q_token=1024, q_head=128, k_token=1024, k_head=128, v_token=1024, v_head=128, qo_token=1024, qo_head=128, tokens=4, q_heads=8,
                               table=P, table_rows=100, rot_dim=128, positions=P, slots=P, cache=cache(), flags=0, stream=None),
    "ztq_kv_read_q8": dict(cache=cache(), slots=P, tokens=4, k_out=P, v_out=P, flags=0, stream=None),
    "ztq_attn_q8": dict(q=P, y=P, q_token=8192, q_head=128, y_token=8192, y_head=128, tokens=4, q_heads=64, query_start=P, kv_len=P, block_table=P, sequences=4, table_width=8, max_new=1,
                        window=0, scale_bits=0x3f800000, cache=cache(), workspace=P, workspace_bytes=1 << 30, flags=0, stream=None),
    "ztq_sample": dict(logits=P, row_stride=1000, rows=4, vocab=1000, temperature=None, top_k=None, top_p=None, min_p=None, uniform=P, token=P, logprob=None, flags=0, stream=None),
}


def call(name, **kw):
    args = CALLS[name] | kw
    assert len(args) == len(_lib.SIGNATURES[name])
    return getattr(_lib.lib(), name)(*[C.addressof(a) if isinstance(a, C.Structure) else a for a in args.values()])


NO_CACHE = [dict(cache=None)] + [dict(cache=cache(**kw)) for kw in (
    dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 4), dict(blocks=0), dict(kv_heads=0), dict(block_size=8), dict(block_size=48), dict(block_size=256),
    dict(head_dim=0), dict(head_dim=100), dict(head_dim=272), dict(block_stride=8 * 16 * 128 - 16), dict(block_stride=8 * 16 * 128 + 8))]
BAD = {
    "ztq_kv_plan": [{n: None} for n in list(CALLS["ztq_kv_plan"])[:12]] + [dict(sequences=0), dict(sequences=4097), dict(table_width=0), dict(block_size=24), dict(block_size=0), dict(pool_blocks=0),
                    dict(max_tokens=0), dict(flags=1), dict(flags=1 << 12), dict(pool_blocks=1 << 27), dict(table_width=1 << 27)],
    "ztq_rope_table": [dict(table=None), dict(table=P + 8), dict(first=-1), dict(rows=0), dict(first=1 << 30, rows=1 << 30), dict(spec=None), dict(flags=2)] + [dict(spec=spec(**kw)) for kw in (
                       dict(rot_dim=8), dict(rot_dim=40), dict(rot_dim=272), dict(base=0), dict(base=float("nan")), dict(base=float("inf")), dict(factor=0), dict(factor=float("inf")), dict(scaling=4),
                       dict(scaling=-1), dict(turns_low=4.0), dict(original_positions=0), dict(magnitude=float("nan")), dict(scaling=3, turns_low=0), dict(scaling=3, base=1.0))],
    "ztq_rope": [dict(x=None), dict(y=None), dict(tokens=-1), dict(heads=0), dict(head_dim=120), dict(head_dim=512), dict(table=None), dict(table=P + 4), dict(table_rows=0), dict(rot_dim=0), dict(rot_dim=24),
                 dict(rot_dim=144), dict(positions=None), dict(flags=4), dict(x=2 * P, y_head=64), dict(x=2 * P, flags=1)],
    "ztq_rope_append_q8": [dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(slots=None), dict(tokens=-1), dict(q_heads=-1), dict(table=P + 4), dict(table_rows=-1), dict(rot_dim=20),
                           dict(rot_dim=160), dict(positions=None), dict(flags=8), dict(q=2 * P, q_token=2048), dict(q=2 * P, flags=2)] + NO_CACHE,
    "ztq_kv_read_q8": [dict(slots=None), dict(tokens=-1), dict(k_out=None, v_out=None), dict(k_out=P + 2), dict(v_out=P + 8), dict(flags=1)] + NO_CACHE,
    "ztq_attn_q8": [{n: None} for n in ("q", "y", "query_start", "kv_len", "block_table", "workspace")] + [
                    dict(tokens=-1), dict(q_heads=0), dict(q_heads=60), dict(sequences=0), dict(sequences=4097), dict(table_width=0), dict(table_width=1 << 27), dict(max_new=0), dict(max_new=1 << 30),
                    dict(window=-1), dict(workspace=P + 8), dict(workspace_bytes=0), dict(workspace_bytes=1000), dict(flags=4), dict(cache=cache(head_dim=32)), dict(cache=cache(head_dim=80))] + NO_CACHE,
    "ztq_sample": [dict(logits=None), dict(uniform=None), dict(token=None), dict(rows=-1), dict(rows=1 << 30), dict(vocab=0), dict(vocab=K.SAMPLE_MAX_VOCAB + 1, row_stride=1 << 20), dict(row_stride=999),
                   dict(flags=2)],
}


@pytest.mark.parametrize("name", list(CALLS))
def test_refusals(name):
    for kw in BAD[name]:
        assert call(name, **kw) == INVALID, kw


@pytest.mark.skipif(torch.cuda.is_available(), reason="the accepted calls would run")
@pytest.mark.parametrize("name", list(CALLS))
def test_the_unchanged_calls_pass_the_checks(name):
    assert call(name) not in (0, INVALID)        # no device here


def test_workspace_of_impossible_sizes_is_zero():
    f = K.attn_q8_workspace_bytes
    assert f(4, 4, 1, 64, 8, 128) > 0
    assert max(f(n * s, s, n, 64, 8, 128) for n in (1, 2, 9, 40, 1000) for s in (1, 2, 5, 18, 19, 64, 500, 4096)) <= 160 << 20
    for bad in ((-1, 4, 1, 64, 8, 128), (4, 0, 1, 64, 8, 128), (4, 4, 0, 64, 8, 128), (4, 4, 1, 63, 8, 128), (4, 4, 1, 64, 0, 128), (4, 4, 1, 64, 8, 100)):
        assert f(*bad) == 0


def test_wrappers_refuse_shapes_types_and_strides():
    """Checked on host tensors: the shape, type and stride tests come before the device's."""
    h = torch.zeros(3, 4, 64, dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    for x in (h.double(), h[0], h.transpose(1, 2)):
        with pytest.raises(ValueError, match="float16 or float32"):
            K._heads(x, "x")
    for t, shape in ((i.long(), (3,)), (i, (4,)), (torch.zeros(6, dtype=torch.int32)[::2], (3,))):
        with pytest.raises(ValueError, match="contiguous torch.int32"):
            K._arg(t, torch.int32, shape, "t")
    with pytest.raises(ValueError, match="scaling"):
        K.rope_table(4, 64, 1e4, scaling="cubic")
    for x in (h, h[0].double(), h[0].t()):
        with pytest.raises(ValueError, match="logits"):
            K.sample(x, i, i)
    k = torch.zeros(5, 2, 16, 64, dtype=torch.int8)
    s = torch.zeros(5, 2)
    for bad in ((k.half(), k, s, s), (k, k[:4], s, s), (k, k.transpose(1, 2), s, s), (k, k, s[:4], s), (k, k, s, s.double())):
        with pytest.raises(ValueError):
            K.KvCache(*bad)
    for args in ((i, None, None), (i, h.double(), None)):
        with pytest.raises(ValueError, match="k_out"):
            K._step().kv_read_q8(0, k, 2, 64, *args, 0, None)
    six = [torch.zeros(6, dtype=torch.int32) for _ in range(12)]
    with pytest.raises(ValueError, match="block_table"):
        K.kv_plan(*six, 16)
    for q, y in ((h, h[:2]), (h[0], h), (h.double(), h)):
        with pytest.raises(ValueError, match="q|y"):
            K._step().attn_q8(q, y, i, i, i, 0, k, 64, i, 1, 1.0, 0, 0, None)
    for q, kk, v in ((None, h, h[:2]), (None, h, h.float()), (h[:2], h, h), (h.float(), h, h)):
        with pytest.raises(ValueError):
            K._step().rope_append_q8(q, kk, v, q, i, 0, k, 4, 64, None, None, 0, None)
    with pytest.raises(ValueError, match="number of arguments"):
        K._step().sample(h)
    with pytest.raises(ValueError, match="a tensor expected"):
        K._step().sample(*[3] * 10)
