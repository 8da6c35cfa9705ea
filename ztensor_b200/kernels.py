"""Python bindings of the C-ABI launchers, one function per kernel.

Same shape as the reference's per-kernel Go wrappers
(internal/cuda/kernels/gemm_q4_purego.go:14, gemm_q8_purego.go,
ternary_gemv_purego.go:19): raw device pointers and ints in, an error out.
Arguments are torch CUDA tensors only so that `.data_ptr()` yields a device
pointer; torch does none of the arithmetic.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

X_F32, Y_F32, X_KB, Y_NB, NO_PDL, PLAIN, FP32_DECODE = 1, 2, 4, 8, 16, 32, 64
FMT_Q4_0, FMT_IQ4NL, FMT_W4G, FMT_Q8_0, FMT_TERNARY = 0, 1, 2, 3, 4


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("kernel arguments must be CUDA tensors (device pointers)")
    return t.data_ptr()


def _stream(stream):
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())     # torch.cuda.current_stream() without its objects
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _stream_arg(stream):
    return stream if stream is None else _stream(stream)


def q4_gpu_data_offset(total_blocks: int) -> int:
    """tensor.Q4GPUDataOffset (tensor/quantized.go:196-199)."""
    return (total_blocks * 2 + 15) & ~15


def gemm_q4_f32(a_q4, b, c, m, k, n, data_offset, stream=None):
    """kernels.GemmQ4F32 (gemm_q4_purego.go:14-29)."""
    _lib.check(_lib.lib().gemm_q4_f32(_ptr(a_q4), _ptr(b), _ptr(c), m, k, n, data_offset, _stream(stream)), "gemm_q4_f32")


def gemm_q8_f32(a_q8, b, c, m, k, n, stream=None):
    """kernels.GemmQ8F32 (gemm_q8_purego.go)."""
    _lib.check(_lib.lib().gemm_q8_f32(_ptr(a_q8), _ptr(b), _ptr(c), m, k, n, _stream(stream)), "gemm_q8_f32")


def ternary_gemv_f32(w, x, y, m, k, stream=None):
    """kernels.TernaryGemvF32 (ternary_gemv_purego.go:19-37)."""
    _lib.check(_lib.lib().ternary_gemv_f32(_ptr(w), _ptr(x), _ptr(y), m, k, _stream(stream)), "ternary_gemv_f32")


def gemv_q4_0(w_sep, data_offset, x, y, n, k, batch, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_q4_0(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)), "ztq_gemv_q4_0")


def gemv_iq4nl(w_sep, data_offset, x, y, n, k, batch, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_iq4nl(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)), "ztq_gemv_iq4nl")


def gemv_q8_0(w, x, y, n, k, batch, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_q8_0(_ptr(w), _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)), "ztq_gemv_q8_0")


def gemv_w4g(qdata, meta, x, y, n, k, group, batch, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_w4g(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, batch, flags, _stream(stream)), "ztq_gemv_w4g")


def gemv_ternary(w_rows, row_scale, x, y, n, k, batch, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_ternary(_ptr(w_rows), _ptr(row_scale), _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)), "ztq_gemv_ternary")


def repack_blocks18(aos, sep, n_blocks, stream=None):
    _lib.check(_lib.lib().ztq_repack_blocks18(_ptr(aos), _ptr(sep), n_blocks, _stream(stream)), "ztq_repack_blocks18")


def pack_w4g_meta(scales, zeros, meta, n_groups, stream=None):
    _lib.check(_lib.lib().ztq_pack_w4g_meta(_ptr(scales), _ptr(zeros), _ptr(meta), n_groups, _stream(stream)), "ztq_pack_w4g_meta")


def repack_ternary_rows(flat, rows, m, k, stream=None):
    _lib.check(_lib.lib().ztq_repack_ternary_rows(_ptr(flat), _ptr(rows), m, k, _stream(stream)), "ztq_repack_ternary_rows")


def quantize_q4_0(src, sep, n, stream=None):
    _lib.check(_lib.lib().ztq_quantize_q4_0(_ptr(src), _ptr(sep), n, _stream(stream)), "ztq_quantize_q4_0")


def quantize_q8_0(src, blocks, n, stream=None):
    _lib.check(_lib.lib().ztq_quantize_q8_0(_ptr(src), _ptr(blocks), n, _stream(stream)), "ztq_quantize_q8_0")


def quantize_w4g(src, qdata, meta, n, group=128, awq=False, stream=None):
    _lib.check(_lib.lib().ztq_quantize_w4g(_ptr(src), _ptr(qdata), _ptr(meta), n, group, 1 if awq else 0, _stream(stream)), "ztq_quantize_w4g")


def dequantize(fmt, w, meta, dst, n, aux, stream=None):
    _lib.check(_lib.lib().ztq_dequantize(fmt, _ptr(w), _ptr(meta), _ptr(dst), n, aux, _stream(stream)), "ztq_dequantize")


def probe_launch(grid, threads, smem_bytes, flags=0, stream=None):
    """An empty kernel with a GEMV's launch shape (the floor of a dependent launch)."""
    _lib.check(_lib.lib().ztq_probe_launch(grid, threads, smem_bytes, flags, _stream(stream)), "ztq_probe_launch")


def check_sm100() -> bool:
    return _lib.lib().ztq_check_sm100() == 1


def device_error() -> int:
    return _lib.lib().ztq_device_error()


def gemv_w4g_allreduce(qdata, meta, x, y, n, k, group, batch, ar, flags=0, stream=None):
    """Row-parallel shard: GEMV + all-reduce of y in one kernel (ar: collective.FusedAllReduce)."""
    _lib.check(_lib.lib().ztq_gemv_w4g_allreduce(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, batch, flags,
                                                 ar.ptr(), _stream(stream)), "ztq_gemv_w4g_allreduce")


def splitk_workspace_bytes(n, splits) -> int:
    return int(_lib.lib().ztq_splitk_workspace_bytes(n, splits))


def gemv_w4g_splitk(qdata, meta, x, y, n, k, group, splits, workspace, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_w4g_splitk(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, splits, _ptr(workspace),
                                              workspace.numel() * workspace.element_size(), flags, _stream(stream)),
               "ztq_gemv_w4g_splitk")


def gemv_q4_0_splitk(w_sep, data_offset, x, y, n, k, splits, workspace, flags=0, stream=None):
    _lib.check(_lib.lib().ztq_gemv_q4_0_splitk(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, splits, _ptr(workspace),
                                               workspace.numel() * workspace.element_size(), flags, _stream(stream)),
               "ztq_gemv_q4_0_splitk")


STATIC_SCRATCH_BYTES = 1 << 20


def gemv_w4g_splitk_static(qdata, meta, x, y, n, k, group, splits, flags=0, stream=None):
    """Split-K GEMV whose partial sums live in the library's built-in scratch array (no workspace argument,
    no allocation; n * splits * 4 <= STATIC_SCRATCH_BYTES; calls must not overlap on the GPU)."""
    _lib.check(_lib.lib().ztq_gemv_w4g_splitk_static(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, splits, flags,
                                                     _stream(stream)), "ztq_gemv_w4g_splitk_static")


def gemm_w4g_tc_workspace_bytes(n, k, batch) -> int:
    return int(_lib.lib().ztq_gemm_w4g_tc_workspace_bytes(n, k, batch))


def gemm_w4g_tc(qdata, meta, x, y, n, k, group, batch, workspace, flags=0, stream=None):
    """W4A16 skinny GEMM on tcgen05 / TMEM (the batch >= 16 path); workspace: uint8 CUDA tensor."""
    _lib.check(_lib.lib().ztq_gemm_w4g_tc(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, batch, _ptr(workspace),
                                          workspace.numel() * workspace.element_size(), flags, _stream(stream)),
               "ztq_gemm_w4g_tc")


def gemm_w4g_tc_allreduce(qdata, meta, x, y, n, k, group, batch, workspace, ar, flags=0, stream=None):
    """Row-parallel shard with 3 or more activation rows: the tensor-core GEMM with the all-reduce of y in its epilogue
    (ar: collective.FusedAllReduce sized for min(batch, 16) * n cells)."""
    _lib.check(_lib.lib().ztq_gemm_w4g_tc_allreduce(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, batch, _ptr(workspace),
                                                    workspace.numel() * workspace.element_size(), flags, ar.ptr(), _stream(stream)),
               "ztq_gemm_w4g_tc_allreduce")


def gemm_q4_0_tc_workspace_bytes(n, k, batch) -> int:
    return int(_lib.lib().ztq_gemm_q4_0_tc_workspace_bytes(n, k, batch))


def gemm_q4_0_tc(w_sep, data_offset, x, y, n, k, batch, workspace, flags=0, stream=None):
    """Q4_0 skinny GEMM on tcgen05 / TMEM (three or more activation rows); workspace: uint8 CUDA tensor."""
    _lib.check(_lib.lib().ztq_gemm_q4_0_tc(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, batch, _ptr(workspace),
                                           workspace.numel() * workspace.element_size(), flags, _stream(stream)),
               "ztq_gemm_q4_0_tc")


def gemm_q8_0_tc_workspace_bytes(n, k, batch) -> int:
    return int(_lib.lib().ztq_gemm_q8_0_tc_workspace_bytes(n, k, batch))


def gemm_q8_0_tc(blocks36, x, y, n, k, batch, workspace, flags=0, stream=None):
    """Q8_0 skinny GEMM on tcgen05 / TMEM (three or more activation rows) on the raw 36-byte blocks."""
    _lib.check(_lib.lib().ztq_gemm_q8_0_tc(_ptr(blocks36), _ptr(x), _ptr(y), n, k, batch, _ptr(workspace),
                                           workspace.numel() * workspace.element_size(), flags, _stream(stream)),
               "ztq_gemm_q8_0_tc")


class ZtqGemvFusion(C.Structure):
    _fields_ = [("residual", C.c_void_p), ("norm_weight", C.c_void_p), ("sum_out", C.c_void_p),
                ("eps_bits", C.c_uint), ("swiglu", C.c_int)]


def gemv_w4g_fused(qdata, meta, x, y, n, k, group=128, flags=0, norm_weight=None, eps=1e-5, residual=None, sum_out=None,
                   swiglu=False, stream=None):
    """Batch-1 W4A16 GEMV with RMSNorm folded into the activation load and / or SwiGLU into the output store."""
    import struct
    fz = ZtqGemvFusion(_ptr(residual), _ptr(norm_weight), _ptr(sum_out),
                       struct.unpack("<I", struct.pack("<f", float(eps)))[0], 1 if swiglu else 0)
    _lib.check(_lib.lib().ztq_gemv_w4g_fused(_ptr(qdata), _ptr(meta), _ptr(x), _ptr(y), n, k, group, flags, C.byref(fz),
                                             _stream(stream)), "ztq_gemv_w4g_fused")


def interleave_rows(a, b, out, rows, row_bytes, stream=None):
    _lib.check(_lib.lib().ztq_interleave_rows(_ptr(a), _ptr(b), _ptr(out), rows, row_bytes, _stream(stream)),
               "ztq_interleave_rows")


def gemv_q4k(w_sep, data_offset, x, y, n, k, batch=1, flags=0, stream=None):
    """Q4_K GEMV on the separated layout of repack_blocks144 (data_offset = 16 * number of super-blocks)."""
    _lib.check(_lib.lib().ztq_gemv_q4k(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)),
               "ztq_gemv_q4k")


def repack_blocks144(aos, sep, nblocks, stream=None):
    _lib.check(_lib.lib().ztq_repack_blocks144(_ptr(aos), _ptr(sep), nblocks, _stream(stream)), "ztq_repack_blocks144")


def gemv_q5k(w_sep, data_offset, x, y, n, k, batch=1, flags=0, stream=None):
    """Q5_K GEMV on the separated layout of repack_blocks176 (data_offset = 48 * number of super-blocks)."""
    _lib.check(_lib.lib().ztq_gemv_q5k(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)),
               "ztq_gemv_q5k")


def repack_blocks176(aos, sep, nblocks, stream=None):
    _lib.check(_lib.lib().ztq_repack_blocks176(_ptr(aos), _ptr(sep), nblocks, _stream(stream)), "ztq_repack_blocks176")


def gemv_q6k(w_sep, data_offset, x, y, n, k, batch=1, flags=0, stream=None):
    """Q6_K GEMV on the separated layout of repack_blocks210 (data_offset = 96 * number of super-blocks)."""
    _lib.check(_lib.lib().ztq_gemv_q6k(_ptr(w_sep), data_offset, _ptr(x), _ptr(y), n, k, batch, flags, _stream(stream)),
               "ztq_gemv_q6k")


def repack_blocks210(aos, sep, nblocks, stream=None):
    _lib.check(_lib.lib().ztq_repack_blocks210(_ptr(aos), _ptr(sep), nblocks, _stream(stream)), "ztq_repack_blocks210")


PLAN_FMT = {"q4_0": 0, "iq4nl": 1, "w4g": 2, "q8_0": 3, "ternary": 4, "q4_k": 5, "q5_k": 6, "q6_k": 7, "w4g_tc": 8}


def describe_plan(fmt: str, n: int, k: int, batch: int = 1, group: int = 128, sms: int = 148) -> dict:
    """The launch plan of the first launch of such a call on a device of `sms` SMs (ztq_describe_plan): host
    arithmetic only, so it also answers without a GPU."""
    out = (C.c_int * 12)()
    if _lib.lib().ztq_describe_plan(PLAN_FMT[fmt], n, k, group, batch, sms, out) != 0:
        raise ValueError(f"no plan for {fmt} {n}x{k} batch {batch}")
    v = list(out)
    if v[0] == 3:
        return dict(kernel="tensor", columns=v[1], k_slices=v[2], groups_per_slice=v[3], row_tiles=v[4], items=v[5],
                    grid=v[6], items_per_cta=v[7])
    return dict(kernel=("plain", "stream", "pair")[v[0]], rows_per_launch=v[1], rt=v[2], rows_per_stage=v[3], stages=v[4],
                overlay_stages=v[5], rows_per_pass=v[6], grid=v[7], tiles_per_cta=v[8], passes_per_cta=v[9],
                warps_per_team=v[10], teams=v[11])


# ---- the decode step around the projections: plan, rotary positions + 8-bit cache, attention, sampling.  Tensors carry
# shapes, strides and types, so these wrappers (the frequent ones in host/ztq_py.cc) check them; X_F32 / Y_F32 follow from the dtypes.

ROPE_PAIRS = 128
ROPE_SCALING = {"none": 0, "linear": 1, "by_turns": 2, "by_dim": 3}
SAMPLE_MAX_VOCAB = 327680


def _arg(t, dtype, shape, name):
    """Device pointer of a contiguous tensor of this type and shape on the current device."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}, strides {t.stride()}")
    return _here(t, name)


def _device():
    try:
        return torch._C._cuda_getDevice()
    except RuntimeError:                        # no device: no tensor is on it
        return -2


def _here(t, name):
    if t.get_device() != _device():
        raise ValueError(f"{name}: a tensor on the current CUDA device expected, got one on {t.device}")
    return t.data_ptr()


def _heads(t, name):
    """(pointer, token stride, head stride, is float32) of a [tokens, heads, dim] tensor with contiguous heads."""
    f32 = t.dtype is torch.float32
    strides = t.stride()
    if len(strides) != 3 or not (f32 or t.dtype is torch.float16) or strides[2] != 1:
        raise ValueError(f"{name}: float16 or float32 [tokens, heads, dim] with contiguous dim expected, got {t.dtype} {tuple(t.shape)}, strides {strides}")
    return _here(t, name), strides[0], strides[1], f32


_native = None


def _step():
    """The native entry points of the operators that a step calls many times (host/ztq_py.cc): checks and launch in one call."""
    global _native
    if _native is None:
        _lib.lib()
        try:
            from . import _step as module
        except ImportError as e:
            raise _lib.KernelLibraryMissing(f"ztensor_b200/_step.so cannot be loaded ({e}): build it with `make -C ztensor_b200/host`") from e
        _native = module
    return _native


class ZtqKvCache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("block_stride", C.c_longlong),
                ("blocks", C.c_int), ("kv_heads", C.c_int), ("block_size", C.c_int), ("head_dim", C.c_int)]


class ZtqRopeSpec(C.Structure):
    _fields_ = [("base", C.c_double), ("factor", C.c_double), ("turns_low", C.c_double), ("turns_high", C.c_double),
                ("original_positions", C.c_double), ("magnitude", C.c_double), ("rot_dim", C.c_int), ("scaling", C.c_int)]


class KvCache:
    """One layer's paged 8-bit cache: k, v int8 [blocks, kv_heads, block_size, head_dim] (the block stride is free, the rest
    contiguous), k_scale, v_scale float32 [blocks, kv_heads].  Keeps the tensors alive and their description ready."""

    def __init__(self, k, v, k_scale, v_scale):
        blocks, heads, size, dim = k.shape
        for t, name in ((k, "k"), (v, "v")):
            if t.dtype is not torch.int8 or t.shape != k.shape or t.stride()[1:] != (size * dim, dim, 1) or t.stride(0) != k.stride(0):
                raise ValueError(f"{name}: int8 [blocks, kv_heads, block_size, head_dim] with contiguous blocks expected, got {t.dtype} {tuple(t.shape)}, strides {t.stride()}")
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _arg(t, torch.float32, (blocks, heads), name)
        self.tensors = (k, v, k_scale, v_scale)
        self.blocks, self.kv_heads, self.block_size, self.head_dim = blocks, heads, size, dim
        self.desc = ZtqKvCache(_here(k, "k"), _here(v, "v"), k_scale.data_ptr(), v_scale.data_ptr(), k.stride(0) if blocks > 1 else heads * size * dim, blocks, heads, size, dim)
        self.ptr = C.addressof(self.desc)
        self.codes = k

    @classmethod
    def empty(cls, blocks, kv_heads, block_size, head_dim, device="cuda"):
        """A cache of its own memory; nothing in it needs a start value."""
        k, v = (torch.empty(blocks, kv_heads, block_size, head_dim, dtype=torch.int8, device=device) for _ in range(2))
        return cls(k, v, *(torch.zeros(blocks, kv_heads, device=device) for _ in range(2)))


def kv_plan(ctx_len, new_len, block_table, ring, ring_state, ring_state_out, next_len, kv_len, query_start, positions, slots, status, block_size, flags=0, stream=None):
    """The plan of a step: block table, slots, positions and lengths from the sequences' lengths (ztq_kv_plan).
    All int32; next_len may be ctx_len and ring_state_out may be ring_state."""
    _step().kv_plan(ctx_len, new_len, block_table, ring, ring_state, ring_state_out, next_len, kv_len, query_start, positions, slots, status, block_size, flags, _stream_arg(stream))


def rope_table(rows, rot_dim, base, first=0, scaling="none", factor=1.0, turns_low=1.0, turns_high=4.0, original_positions=0, magnitude=1.0, out=None, flags=0, stream=None):
    """{cos, sin} of positions first .. first + rows - 1, float32 [rows, rot_dim / 2, 2] (ztq_rope_table)."""
    if scaling not in ROPE_SCALING:
        raise ValueError(f"scaling: one of {sorted(ROPE_SCALING)} expected, got {scaling!r}")
    if out is None:
        out = torch.empty(rows, rot_dim // 2, 2, dtype=torch.float32, device="cuda")
    spec = ZtqRopeSpec(base, factor, turns_low, turns_high, original_positions, magnitude, rot_dim, ROPE_SCALING[scaling])
    _lib.check(_lib.lib().ztq_rope_table(_arg(out, torch.float32, (rows, rot_dim // 2, 2), "out"), first, rows, C.addressof(spec), flags, _stream(stream)), "ztq_rope_table")
    return out


def rope(x, y, table, positions, flags=0, stream=None):
    """y = x [tokens, heads, dim] rotated to `positions`; y may be x (ztq_rope)."""
    xp, xt, xh, xf = _heads(x, "x")
    yp, yt, yh, yf = _heads(y, "y")
    n, heads, dim = x.shape
    if y.shape != x.shape:
        raise ValueError(f"y: {tuple(x.shape)} expected, got {tuple(y.shape)}")
    _lib.check(_lib.lib().ztq_rope(xp, yp, n, heads, dim, xt, xh, yt, yh, _arg(table, torch.float32, (*table.shape[:2], 2), "table"), table.shape[0], 2 * table.shape[1],
                                   _arg(positions, torch.int32, (n,), "positions"), flags | (X_F32 if xf else 0) | (Y_F32 if yf else 0), _stream(stream)), "ztq_rope")


def rope_append_q8(q, k, v, q_out, slots, cache, table=None, positions=None, flags=0, stream=None):
    """Rotates q [tokens, q_heads, dim] into q_out (both may be None, or q_out may be q) and appends k (rotated), v [tokens, kv_heads, dim] to
    the cache at `slots` (ztq_rope_append_q8).  table None: nothing is rotated.  flags: ROPE_PAIRS, NO_PDL."""
    _step().rope_append_q8(q, k, v, q_out, slots, cache.ptr, cache.codes, cache.kv_heads, cache.head_dim, table, positions, flags, _stream_arg(stream))


def kv_read_q8(cache, slots, k_out, v_out, flags=0, stream=None):
    """The cache's rows at `slots`, dequantized into k_out and v_out [tokens, kv_heads, dim] (either may be None) (ztq_kv_read_q8)."""
    _step().kv_read_q8(cache.ptr, cache.codes, cache.kv_heads, cache.head_dim, slots, k_out, v_out, flags, _stream_arg(stream))


def attn_q8_workspace_bytes(tokens, sequences, max_new, q_heads, kv_heads, head_dim) -> int:
    return int(_lib.lib().ztq_attn_q8_workspace_bytes(tokens, sequences, max_new, q_heads, kv_heads, head_dim))


def attn_q8(q, y, query_start, kv_len, block_table, cache, workspace, max_new, scale, window=0, flags=0, stream=None):
    """Causal attention of q [tokens, q_heads, dim] over the cache into y (ztq_attn_q8); window 0: all earlier positions."""
    _step().attn_q8(q, y, query_start, kv_len, block_table, cache.ptr, cache.codes, cache.head_dim, workspace, max_new, scale, window, flags, _stream_arg(stream))


def sample(logits, uniform, token, logprob=None, temperature=None, top_k=None, top_p=None, min_p=None, flags=0, stream=None):
    """One token per row of logits [rows, vocab] from `uniform` [rows] in [0, 1) (ztq_sample)."""
    _step().sample(logits, uniform, token, logprob, temperature, top_k, top_p, min_p, flags, _stream_arg(stream))
