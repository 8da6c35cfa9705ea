// ztq_lib.cu -- the extern "C" launchers of libztq_sm100a.so (see include/ztq.h).
//
// Host side of every launcher: validate, derive the launch plan from the shape
// alone (no state is kept between calls, so calls from any thread are safe),
// launch asynchronously on the caller's stream, return cudaGetLastError().
#include "../../include/ztq.h"

#include "formats.cuh"
#include "gemv_stream.cuh"
#include "gemv_w4pair.cuh"
#include "gemm_w4g_tc.cuh"
#include "launch.cuh"
#include "ztq_common.cuh"

#include <atomic>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <mutex>
#include <vector>

namespace ztq {

// ---------------------------------------------------------------------------
// Launch plan of the streaming GEMV.
// ---------------------------------------------------------------------------
struct Plan {
    bool ok = false;
    int spt = 1;
    int rt = 2;
    bool big = false;
    bool fp = false;          // fp32 decode instead of the integer inner loop
    int threads = 0;
    int grid = 0;
    size_t smem = 0;
    GemvParams p;
};

// slot_w: weights per lane per row (the format's natural slot, or 64 for the
// chunk-pair kernel).
template <int FMT>
static Plan make_plan(GemvParams p, int batch_chunk, const DeviceInfo& dev, int slot_w = FmtTraits<FMT>::SLOT_W) {
    using TR = FmtTraits<FMT>;
    Plan pl;
    const bool pair = slot_w != TR::SLOT_W;
    if (p.K % slot_w) return pl;
    p.slots = p.K / slot_w;
    if (p.row_bytes % 16 || p.meta_row_bytes % 16) return pl;       // bulk copies move whole 16-byte units
    if ((reinterpret_cast<uintptr_t>(p.w) & 15) || (reinterpret_cast<uintptr_t>(p.meta) & 15)) return pl;
    // Slots per thread: one while a team of <= 8 warps spans K, two for longer rows
    // (only with a single activation vector and 32-wide slots: register budget).
    const bool can2 = (batch_chunk == 1) && (TR::SLOT_W == 32);
    int spt = 1;
    int wpt = ceil_div(p.slots, 32);
    if (wpt > 8 && !pair) {
        if (!can2) return pl;
        spt = 2;
        wpt = ceil_div(p.slots, 64);
    }
    if (wpt > 16) return pl;
    if (pair && p.slots < 32) return pl;                  // short rows: the one-chunk kernel keeps all lanes busy
    const bool big = wpt > 8;
    const int teams = big ? 1 : 8 / wpt;
    p.WPT = wpt;
    p.T = teams;
    // rows per team per stage: 4 while a stage stays below 40 KB (two stages still fit half an SM), else 2
    const int rb = p.row_bytes + p.meta_row_bytes;
    int rt = (spt == 1 && !big && teams * 4 * rb <= 40 * 1024 && batch_chunk * 4 <= 8) ? 4 : 2;   // spt 2 / big: RT = 2 only
    p.R = teams * rt;
    const int cw = teams * wpt;
    const int stage = p.R * rb;
    p.stage_stride = (stage + 127) & ~127;
    // partial sums of one pass: [P rows][BC][WPT] floats
    const int rows_per_cta = ceil_div(p.N, dev.sms > 0 ? dev.sms : 1);
    int P = ceil_div(rows_per_cta, p.R) * p.R;
    const int p_max = (24 * 1024 / (4 * batch_chunk * wpt)) / p.R * p.R;
    if (P > p_max) P = p_max;
    if (P < p.R) return pl;
    p.P = P;
    const int part_bytes = P * batch_chunk * wpt * 4 + (FMT == F_IQ4NL ? 2048 : 0);
    const int budget = (big ? 216 : 108) * 1024 - part_bytes - 512;
    int S = budget / p.stage_stride;
    if (S < 2) return pl;
    if (S > 16) S = 16;
    p.S = S;
    p.part_off = S * p.stage_stride;
    p.bar_off = (p.part_off + part_bytes + 15) & ~15;
    pl.smem = (size_t)p.bar_off + 2 * S * 8 + 16;
    pl.threads = (cw + 1) * 32;
    const long long tiles = ceil_div(p.N, p.R);
    // two co-resident CTAs per SM unless one owns it; a small problem takes one slot per SM and leaves the
    // other to the next kernel of the stream (programmatic dependent launch), which prefetches meanwhile
    const bool small = false;   // one CTA per SM for small problems measured slower
    long long grid = (long long)dev.sms * ((big || small) ? 1 : 2);
    if (grid > tiles) grid = tiles;
    if (grid < 1) grid = 1;
    pl.grid = (int)grid;
    pl.spt = spt;
    pl.rt = rt;
    pl.big = big;
    pl.p = p;
    pl.ok = true;
    return pl;
}

template <int FMT, int BC, int SPT, int RT, bool BIG, bool FP, bool AR = false>
static cudaError_t launch_stream_inst2(const Plan& pl, cudaStream_t stream, bool pdl) {
    auto kern = gemv_stream_kernel<FMT, BC, SPT, RT, BIG, FP, AR>;
    // One-time opt-in to large dynamic shared memory, per kernel and device.
    static std::atomic<unsigned> done_mask{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned bit = 1u << (dev & 31);
    if (!(done_mask.load(std::memory_order_acquire) & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        done_mask.fetch_or(bit, std::memory_order_release);
    }
    return launch(kern, dim3(pl.grid), dim3(pl.threads), pl.smem, stream, pdl, pl.p);
}

template <int FMT, int BC, int SPT, int RT, bool BIG>
static cudaError_t launch_stream_inst(const Plan& pl, cudaStream_t stream, bool pdl) {
    if (pl.p.ar.world > 1) {
        // the all-reduce instantiations: the two formats with an *_allreduce entry point, integer inner loop
        if constexpr (FMT == F_W4G || FMT == F_Q4_0) {
            if (!pl.fp) return launch_stream_inst2<FMT, BC, SPT, RT, BIG, false, true>(pl, stream, pdl);
        }
        return cudaErrorInvalidValue;
    }
    if (pl.fp || FMT == F_IQ4NL) return launch_stream_inst2<FMT, BC, SPT, RT, BIG, true>(pl, stream, pdl);
    if constexpr (FMT != F_IQ4NL) return launch_stream_inst2<FMT, BC, SPT, RT, BIG, false>(pl, stream, pdl);
    return cudaErrorInvalidValue;
}

template <int FMT, int BC>
static cudaError_t launch_stream(const Plan& pl, cudaStream_t stream, bool pdl) {
    if (pl.big) {
        if (pl.spt == 2) { if constexpr (BC == 1 && FMT != F_TERN) return launch_stream_inst<FMT, 1, 2, 2, true>(pl, stream, pdl); }
        return cudaErrorInvalidValue;
    }
    if (pl.spt == 2) {
        if constexpr (BC == 1 && FMT != F_TERN) return launch_stream_inst<FMT, 1, 2, 2, false>(pl, stream, pdl);
        return cudaErrorInvalidValue;
    }
    if (pl.rt == 4) return launch_stream_inst<FMT, BC, 1, 4, false>(pl, stream, pdl);
    return launch_stream_inst<FMT, BC, 1, 2, false>(pl, stream, pdl);
}

// Plan of the chunk-pair kernel: one CTA per SM, up to 16 consumer warps, the
// converted activations (3 K + K/4 bytes) in shared memory next to the stages.
template <int FMT>
static Plan make_pair_plan(GemvParams p, const DeviceInfo& dev) {
    Plan pl;
    if (p.K % 64) return pl;
    p.slots = p.K / 64;
    if (p.slots < 32) return pl;
    if (p.row_bytes % 16 || p.meta_row_bytes % 16) return pl;
    if ((reinterpret_cast<uintptr_t>(p.w) & 15) || (reinterpret_cast<uintptr_t>(p.meta) & 15)) return pl;
    const int wpt = ceil_div(p.slots, 32);
    if (wpt > 16) return pl;
    const int rb = p.row_bytes + p.meta_row_bytes;
    const int rows_per_cta = ceil_div(p.N, dev.sms > 0 ? dev.sms : 1);
    // Small share per CTA (it fits a few stages): 8 consumer warps and half an SM, so that the next kernel of
    // the stream (programmatic dependent launch) is resident beside this one and has its weights in shared
    // memory by the time this one finishes.  Large share: 16 consumer warps, the whole SM, a deep ring.
    // (a half-SM variant with 8 consumer warps, meant to let the next kernel prefetch beside this one, measured
    // slower on every shape: the conversion and the compute lose more than the overlap gains)
    const bool small = false;
    const int teams = (small ? 8 : 16) / wpt;
    p.WPT = wpt;
    p.T = teams;
    // Rows per team per stage: four when that still leaves (nearly) every SM a tile and two stages fit -- the
    // per-stage costs (barrier round trip, butterfly, partial-sum stores) are then shared by twice the rows, which
    // measured 4-9 % faster -- else two.
    for (int rt = 4; rt >= 2; rt -= 2) {
        if (rt == 4 && ceil_div(p.N, teams * 4) * 5 < (long long)dev.sms * 4) continue;
        p.R = teams * rt;
        p.stage_stride = (p.R * rb + 127) & ~127;
        int P = ceil_div(rows_per_cta, p.R) * p.R;
        const int p_max = (16 * 1024 / (4 * wpt)) / p.R * p.R;
        if (P > p_max) P = p_max;
        if (P < p.R) continue;
        p.P = P;
        const int part_bytes = P * wpt * 4;
        const int x_bytes = 3 * p.K + (p.K / 64) * 16;
        const int budget = 220 * 1024 - part_bytes - x_bytes - 1024;
        int S = budget / p.stage_stride;
        if (S < 2) continue;
        if (S > 12) S = 12;
        p.S = S;
        p.x_off = S * p.stage_stride;
        p.part_off = (p.x_off + x_bytes + 15) & ~15;
        p.bar_off = (p.part_off + part_bytes + 15) & ~15;
        p.Sx = (p.part_off - p.x_off) / p.stage_stride;       // stages that fit where the activation planes were
        pl.smem = (size_t)p.bar_off + 2 * (S + p.Sx) * 8 + 8 + 16;
        pl.threads = (teams * wpt + 1) * 32;
        const long long tiles = ceil_div(p.N, p.R);
        long long grid = dev.sms;
        if (grid > tiles) grid = tiles;
        pl.grid = (int)(grid < 1 ? 1 : grid);
        pl.rt = rt;
        pl.p = p;
        pl.ok = true;
        return pl;
    }
    return pl;
}

template <int FMT, int RT, bool FUSED = false, bool AR = false>
static cudaError_t launch_pair_inst(const Plan& pl, cudaStream_t stream, bool pdl) {
    auto kern = gemv_w4pair_kernel<FMT, RT, FUSED, AR>;
    static std::atomic<unsigned> done_mask{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned bit = 1u << (dev & 31);
    if (!(done_mask.load(std::memory_order_acquire) & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        done_mask.fetch_or(bit, std::memory_order_release);
    }
    return launch(kern, dim3(pl.grid), dim3(pl.threads), pl.smem, stream, pdl, pl.p);
}

template <int FMT>
static cudaError_t launch_pair(const Plan& pl, cudaStream_t stream, bool pdl) {
    if (pl.p.ar.world > 1) {
        if constexpr (FMT == F_W4G || FMT == F_Q4_0)
            return pl.rt == 4 ? launch_pair_inst<FMT, 4, false, true>(pl, stream, pdl) : launch_pair_inst<FMT, 2, false, true>(pl, stream, pdl);
        return cudaErrorInvalidValue;
    }
    return pl.rt == 4 ? launch_pair_inst<FMT, 4>(pl, stream, pdl) : launch_pair_inst<FMT, 2>(pl, stream, pdl);
}

template <int FMT>
static cudaError_t launch_plain(GemvParams p, int batch, cudaStream_t stream, bool pdl) {
    using TR = FmtTraits<FMT>;
    if (p.K % TR::SLOT_W) return cudaErrorInvalidValue;
    p.slots = p.K / TR::SLOT_W;
    const int wpb = 8;
    return launch(gemv_plain_kernel<FMT>, dim3(ceil_div(p.N, wpb)), dim3(wpb * 32), 0, stream, pdl, p, batch);
}

// y[b, n] for b in [0, batch): chunks of two activation vectors per launch of
// the streaming kernel (one for ternary and for rows too long to keep two
// vectors in registers).
template <int FMT>
static cudaError_t gemv_dispatch(GemvParams p, int batch, int flags, cudaStream_t stream) {
    if (p.N <= 0 || p.K <= 0 || batch <= 0) return cudaErrorInvalidValue;
    if (!p.w || !p.x || !p.y) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    const bool pdl = !(flags & ZTQ_NO_PDL);
    p.x_f32 = (flags & ZTQ_X_F32) ? 1 : 0;
    p.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
    if (flags & ZTQ_X_KB) { p.xs_b = 1; p.xs_k = batch; } else { p.xs_b = p.K; p.xs_k = 1; }
    if (flags & ZTQ_Y_NB) { p.ys_b = 1; p.ys_n = batch; } else { p.ys_b = p.N; p.ys_n = 1; }

    const int max_bc = (FMT == F_TERN) ? 1 : 2;
    Plan pl2, pl1, plp;
    if (!(flags & ZTQ_PLAIN)) {
        if (max_bc == 2) pl2 = make_plan<FMT>(p, 2, dev);
        pl1 = make_plan<FMT>(p, 1, dev);
        // the chunk-pair kernel pays for its shared activation planes with a longer prologue: with fewer than a
        // dozen rows per SM the one-chunk kernel is ahead (1280 x 8192: 4.3 against 5.1 us)
        if ((FMT == F_Q4_0 || (FMT == F_W4G && p.gshift == 2)) && !(flags & ZTQ_FP32_DECODE) && (p.ys_n == 1 || batch == 1) &&
            (long long)p.N >= 12LL * dev.sms)
            plp = make_pair_plan<FMT>(p, dev);
    }
    if (!pl1.ok) {
        if (p.ar.world > 1) return cudaErrorInvalidValue;      // the fused all-reduce lives in the streaming kernels
        return launch_plain<FMT>(p, batch, stream, pdl);
    }

    const size_t xe = p.x_f32 ? 4 : 2, ye = p.y_f32 ? 4 : 2;
    int b = 0;
    while (b < batch) {
        const bool two = (batch - b >= 2) && pl2.ok && pl2.spt == 1;
        Plan pl = two ? pl2 : pl1;
        pl.fp = (flags & ZTQ_FP32_DECODE) != 0;
        pl.p.x = static_cast<const uint8_t*>(p.x) + (size_t)b * p.xs_b * xe;
        pl.p.y = static_cast<uint8_t*>(p.y) + (size_t)b * p.ys_b * ye;
        cudaError_t e;
        if (!two && plp.ok) {
            if constexpr (FMT == F_Q4_0 || FMT == F_W4G) {
                Plan pp = plp;
                pp.p.x = pl.p.x;
                pp.p.y = pl.p.y;
                e = launch_pair<FMT>(pp, stream, pdl);
            } else e = cudaErrorInvalidValue;
        } else if (two) {
            if constexpr (FMT == F_TERN) e = cudaErrorInvalidValue;
            else e = launch_stream<FMT, 2>(pl, stream, pdl);
        } else e = launch_stream<FMT, 1>(pl, stream, pdl);
        if (e != cudaSuccess) return e;
        b += two ? 2 : 1;
    }
    return cudaGetLastError();
}

}  // namespace ztq

// ---- split-K -----------------------------------------------------------------
// Narrow outputs (few rows, long K): the grid is split along K, every split writes fp32 partial sums of all N
// rows to the workspace, a second kernel adds the splits in order.  Deterministic: no atomics.
namespace ztq {
template <int FMT>
static cudaError_t gemv_splitk(GemvParams p, int splits, int group, void* workspace, size_t workspace_bytes, int flags,
                               cudaStream_t stream) {
    if (p.N <= 0 || p.K <= 0 || splits < 2 || splits > 64 || !p.w || !p.x || !p.y || !workspace) return cudaErrorInvalidValue;
    if (workspace_bytes < (size_t)splits * p.N * 4 || (reinterpret_cast<uintptr_t>(workspace) & 15)) return cudaErrorInvalidValue;
    // contiguous [1, K] activations and [1, N] outputs only: the layout flags of the GEMV entry points do not apply
    if (flags & ~(ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_NO_PDL | ZTQ_FP32_DECODE)) return cudaErrorInvalidValue;
    if (p.K % splits) return cudaErrorInvalidValue;
    const int kc = p.K / splits;
    if (kc % 32 || (FMT == F_W4G && kc % group)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    const bool pdl = !(flags & ZTQ_NO_PDL);
    GemvParams c = p;                                  // one split: K/splits columns of every row
    c.w_stride = p.row_bytes;
    c.meta_stride = p.meta_row_bytes;
    c.K = kc;
    c.row_bytes = p.row_bytes / splits;
    c.meta_row_bytes = p.meta_row_bytes / splits;
    c.splits = splits;
    c.x_f32 = (flags & ZTQ_X_F32) ? 1 : 0;
    c.y_f32 = 1;                                       // partial sums are fp32
    c.xs_b = p.K; c.xs_k = 1; c.ys_b = p.N; c.ys_n = 1;
    c.y = workspace;
    Plan pl = make_plan<FMT>(c, 1, dev);
    if (!pl.ok || pl.spt != 1 || pl.big) return cudaErrorInvalidValue;   // slices must fit the one-slot kernel
    const int tiles = ceil_div(p.N, pl.p.R);
    int per_split = ceil_div(2 * dev.sms, splits);
    if (per_split > tiles) per_split = tiles;
    if (per_split < 1) per_split = 1;
    pl.grid = per_split * splits;
    pl.fp = (flags & ZTQ_FP32_DECODE) != 0;
    cudaError_t e = launch_stream<FMT, 1>(pl, stream, pdl);
    if (e != cudaSuccess) return e;
    e = launch(splitk_reduce_kernel, dim3(ceil_div(p.N, 256)), dim3(256), 0, stream, pdl,
               static_cast<const float*>(workspace), p.y, p.N, splits, (flags & ZTQ_Y_F32) ? 1 : 0);
    return e != cudaSuccess ? e : cudaGetLastError();
}
}  // namespace ztq

namespace ztq {
// Q4_K / Q5_K: side bytes per super-block (header, plus qh for Q5_K) first, nibbles at data_offset
template <int FMT>
static cudaError_t gemv_kquant(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch,
                               int flags, cudaStream_t stream) {
    constexpr int SIDE = FMT == F_Q6K ? 96 : FMT == F_Q5K ? 48 : 16;
    if (!w_sep || !x || !y || N <= 0 || K <= 0 || batch <= 0 || batch > 8) return cudaErrorInvalidValue;
    if (K % 256 || data_offset <= 0 || (data_offset & 15) || (reinterpret_cast<uintptr_t>(w_sep) & 15)) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_NO_PDL)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    GemvParams p = {};
    p.meta = static_cast<const uint8_t*>(w_sep);
    p.w = p.meta + data_offset;
    p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = K / 256 * SIDE;
    p.x_f32 = (flags & ZTQ_X_F32) ? 1 : 0;
    p.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
    p.xs_b = K; p.xs_k = 1; p.ys_b = N; p.ys_n = 1;
    p.x = x; p.y = y;
    Plan pl = make_pair_plan<FMT>(p, dev);
    if (!pl.ok) return cudaErrorInvalidValue;                 // rows shorter than 2048 are not taken
    const size_t xe = p.x_f32 ? 4 : 2, ye = p.y_f32 ? 4 : 2;
    for (int b = 0; b < batch; ++b) {                         // one pass per activation row
        pl.p.x = static_cast<const uint8_t*>(x) + (size_t)b * K * xe;
        pl.p.y = static_cast<uint8_t*>(y) + (size_t)b * N * ye;
        cudaError_t e = launch_pair<FMT>(pl, stream, !(flags & ZTQ_NO_PDL));
        if (e != cudaSuccess) return e;
    }
    return cudaGetLastError();
}

}  // namespace ztq

using namespace ztq;

extern "C" {
int ztq_take_error_step();
int ztq_take_error_attn();
}

// ---- batch >= 16: W4A16 skinny GEMM on tcgen05 / TMEM -------------------------------
namespace {
template <int NB, bool I8, bool SPLIT, int GB = 1, bool AR = false, bool W8 = false>
cudaError_t launch_tc(const CUtensorMap& map, const TcParams& tp, int grid, size_t smem, cudaStream_t stream, bool pdl) {
    auto kern = gemm_w4g_tc_kernel<NB, I8, SPLIT, GB, AR, W8>;
    static std::atomic<unsigned> done_mask{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned bit = 1u << (dev & 31);
    if (!(done_mask.load(std::memory_order_acquire) & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        done_mask.fetch_or(bit, std::memory_order_release);
    }
    return launch(kern, dim3(grid), dim3(kTcThreads), smem, stream, pdl, map, tp);
}
}  // namespace


// group sizes: powers of two from 32 up (32-weight slots must not straddle a group)
static int group_shift(int group) {
    for (int s = 0; s < 12; ++s)
        if (group == (32 << s)) return s;
    return -1;
}


// ===========================================================================
// extern "C"
// ===========================================================================
extern "C" {

cudaError_t ztq_gemv_q4_0(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch,
                          int flags, cudaStream_t stream) {
    if (!w_sep || K % 32 || data_offset < 0 || (data_offset & 15)) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.meta = static_cast<const uint8_t*>(w_sep);
    p.w = p.meta + data_offset;
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = K / 16;
    return gemv_dispatch<F_Q4_0>(p, batch, flags, stream);
}

cudaError_t ztq_gemv_iq4nl(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch,
                           int flags, cudaStream_t stream) {
    if (!w_sep || K % 32 || data_offset < 0 || (data_offset & 15)) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.meta = static_cast<const uint8_t*>(w_sep);
    p.w = p.meta + data_offset;
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = K / 16;
    return gemv_dispatch<F_IQ4NL>(p, batch, flags, stream);
}

cudaError_t ztq_gemv_q8_0(const void* w_blocks36, const void* x, void* y, int N, int K, int batch, int flags,
                          cudaStream_t stream) {
    if (K % 32) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.w = static_cast<const uint8_t*>(w_blocks36);
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = (K / 32) * 36;
    p.meta_row_bytes = 0;
    return gemv_dispatch<F_Q8_0>(p, batch, flags, stream);
}

cudaError_t ztq_gemv_w4g(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                         int batch, int flags, cudaStream_t stream) {
    const int gs = group_shift(group);
    if (gs < 0 || K % group || !meta) return cudaErrorInvalidValue;       // groups must not straddle rows
    GemvParams p = {};
    p.w = static_cast<const uint8_t*>(qdata);
    p.meta = static_cast<const uint8_t*>(meta);
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = (K / group) * 4;
    p.gshift = gs;
    return gemv_dispatch<F_W4G>(p, batch, flags, stream);
}

cudaError_t ztq_gemv_ternary(const void* w_rows, const void* row_scale, const void* x, void* y, int N, int K,
                             int batch, int flags, cudaStream_t stream) {
    if (K % 64) return cudaErrorInvalidValue;    // 128-bit loads; other K go through ternary_gemv_f32
    GemvParams p = {};
    p.w = static_cast<const uint8_t*>(w_rows);
    p.row_scale = static_cast<const __half*>(row_scale);
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 4;
    p.meta_row_bytes = 0;
    return gemv_dispatch<F_TERN>(p, batch, flags, stream);
}

cudaError_t ztq_gemv_q4k(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch, int flags,
                         cudaStream_t stream) {
    return gemv_kquant<F_Q4K>(w_sep, data_offset, x, y, N, K, batch, flags, stream);
}
cudaError_t ztq_gemv_q5k(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch, int flags,
                         cudaStream_t stream) {
    return gemv_kquant<F_Q5K>(w_sep, data_offset, x, y, N, K, batch, flags, stream);
}

cudaError_t ztq_gemv_q6k(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch, int flags,
                         cudaStream_t stream) {
    return gemv_kquant<F_Q6K>(w_sep, data_offset, x, y, N, K, batch, flags, stream);
}

cudaError_t ztq_repack_blocks210(const void* aos, void* sep, long long nblocks, cudaStream_t stream) {
    if (!aos || !sep || nblocks <= 0 || (reinterpret_cast<uintptr_t>(sep) & 15)) return cudaErrorInvalidValue;
    long long blocks = ceil_div(nblocks * 14, 256);
    if (blocks > 65535) blocks = 65535;
    repack_blocks210_kernel<<<(unsigned)blocks, 256, 0, stream>>>(static_cast<const uint8_t*>(aos), static_cast<uint8_t*>(sep),
                                                                  nblocks, nblocks * 96);
    return cudaGetLastError();
}

cudaError_t ztq_repack_blocks176(const void* aos, void* sep, long long nblocks, cudaStream_t stream) {
    if (!aos || !sep || nblocks <= 0) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(aos) | reinterpret_cast<uintptr_t>(sep)) & 15) return cudaErrorInvalidValue;
    long long blocks = ceil_div(nblocks * 11, 256);
    if (blocks > 65535) blocks = 65535;
    repack_blocks176_kernel<<<(unsigned)blocks, 256, 0, stream>>>(static_cast<const uint8_t*>(aos), static_cast<uint8_t*>(sep),
                                                                  nblocks, nblocks * 48);
    return cudaGetLastError();
}

cudaError_t ztq_repack_blocks144(const void* aos, void* sep, long long nblocks, cudaStream_t stream) {
    if (!aos || !sep || nblocks <= 0) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(aos) | reinterpret_cast<uintptr_t>(sep)) & 15) return cudaErrorInvalidValue;
    long long blocks = ceil_div(nblocks * 9, 256);
    if (blocks > 65535) blocks = 65535;
    repack_blocks144_kernel<<<(unsigned)blocks, 256, 0, stream>>>(static_cast<const uint8_t*>(aos), static_cast<uint8_t*>(sep),
                                                                  nblocks, nblocks * 16);
    return cudaGetLastError();
}

cudaError_t ztq_gemv_w4g_fused(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group, int flags,
                               const ZtqGemvFusion* fz, cudaStream_t stream) {
    if (!qdata || !meta || !x || !y || !fz || N <= 0 || K <= 0 || group != 128 || K % 256) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_NO_PDL)) return cudaErrorInvalidValue;
    if (fz->swiglu && (N & 1)) return cudaErrorInvalidValue;
    if (fz->norm_weight && (reinterpret_cast<uintptr_t>(fz->norm_weight) & 15)) return cudaErrorInvalidValue;
    if (!fz->norm_weight && (fz->residual || fz->sum_out)) return cudaErrorInvalidValue;   // they belong to the RMSNorm
    if (fz->sum_out && (fz->sum_out == x || fz->sum_out == fz->residual)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    GemvParams p = {};
    p.w = static_cast<const uint8_t*>(qdata);
    p.meta = static_cast<const uint8_t*>(meta);
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = (K / group) * 4;
    p.gshift = 2;
    p.x_f32 = (flags & ZTQ_X_F32) ? 1 : 0;
    p.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
    p.xs_b = K; p.xs_k = 1; p.ys_b = fz->swiglu ? N / 2 : N; p.ys_n = 1;
    p.fz.residual = fz->residual;
    p.fz.norm_weight = static_cast<const float*>(fz->norm_weight);
    p.fz.sum_out = fz->sum_out;
    std::memcpy(&p.fz.eps, &fz->eps_bits, 4);
    p.fz.swiglu = fz->swiglu ? 1 : 0;
    const Plan pl = make_pair_plan<F_W4G>(p, dev);
    if (!pl.ok) return cudaErrorInvalidValue;                 // the fusions live in the chunk-pair kernel (K >= 2048)
    return pl.rt == 4 ? launch_pair_inst<F_W4G, 4, true>(pl, stream, !(flags & ZTQ_NO_PDL))
                      : launch_pair_inst<F_W4G, 2, true>(pl, stream, !(flags & ZTQ_NO_PDL));
}

cudaError_t ztq_interleave_rows(const void* a, const void* b, void* out, long long rows, int row_bytes, cudaStream_t stream) {
    if (!a || !b || !out || rows <= 0 || row_bytes <= 0 || row_bytes % 16) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(out)) & 15) return cudaErrorInvalidValue;
    const long long total = rows * (row_bytes / 16);
    long long blocks = ceil_div(total, 256);
    if (blocks > 65535) blocks = 65535;
    interleave_rows_kernel<<<(unsigned)blocks, 256, 0, stream>>>(static_cast<const uint4*>(a), static_cast<const uint4*>(b),
                                                                 static_cast<uint4*>(out), rows, row_bytes / 16);
    return cudaGetLastError();
}

static cudaError_t fill_ar(GemvParams& p, const ZtqAllReduce* ar, int batch) {
    if (!ar) return cudaSuccess;
    if (ar->world < 2 || ar->world > kMaxRanks || ar->rank < 0 || ar->rank >= ar->world) return cudaErrorInvalidValue;
    if ((long long)batch * p.N > ar->slot_stride || !ar->state) return cudaErrorInvalidValue;
    p.ar.world = ar->world;
    p.ar.rank = ar->rank;
    p.ar.slot_stride = ar->slot_stride;
    for (int r = 0; r < ar->world; ++r) {
        if (!ar->slots[r] || (reinterpret_cast<uintptr_t>(ar->slots[r]) & 7)) return cudaErrorInvalidValue;
        p.ar.slots[r] = static_cast<uint2*>(ar->slots[r]);
    }
    p.ar.state = static_cast<unsigned*>(ar->state);
    return cudaSuccess;
}

cudaError_t ztq_gemv_w4g_allreduce(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                                   int batch, int flags, const ZtqAllReduce* ar, cudaStream_t stream) {
    const int gs = group_shift(group);
    if (gs < 0 || K % group || !meta) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.w = static_cast<const uint8_t*>(qdata);
    p.meta = static_cast<const uint8_t*>(meta);
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = (K / group) * 4;
    p.gshift = gs;
    cudaError_t e = fill_ar(p, ar, batch);
    if (e != cudaSuccess) return e;
    return gemv_dispatch<F_W4G>(p, batch, flags, stream);
}

cudaError_t ztq_gemv_q4_0_allreduce(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch,
                                    int flags, const ZtqAllReduce* ar, cudaStream_t stream) {
    if (!w_sep || K % 32 || data_offset < 0 || (data_offset & 15)) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.meta = static_cast<const uint8_t*>(w_sep);
    p.w = p.meta + data_offset;
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = K / 16;
    cudaError_t e = fill_ar(p, ar, batch);
    if (e != cudaSuccess) return e;
    return gemv_dispatch<F_Q4_0>(p, batch, flags, stream);
}

cudaError_t ztq_symm_alloc(void** ptr, size_t bytes) {
    if (!ptr || bytes == 0) return cudaErrorInvalidValue;
    cudaError_t e = cudaMalloc(ptr, bytes);
    if (e != cudaSuccess) return e;
    return cudaMemset(*ptr, 0, bytes);
}
cudaError_t ztq_symm_free(void* ptr) { return cudaFree(ptr); }
cudaError_t ztq_symm_zero(void* ptr, size_t bytes) {
    if (!ptr || bytes == 0) return cudaErrorInvalidValue;
    cudaError_t e = cudaMemset(ptr, 0, bytes);
    return e != cudaSuccess ? e : cudaDeviceSynchronize();
}
cudaError_t ztq_ipc_export(void* ptr, void* handle64) {
    if (!ptr || !handle64) return cudaErrorInvalidValue;
    static_assert(sizeof(cudaIpcMemHandle_t) == 64, "handle size");
    return cudaIpcGetMemHandle(static_cast<cudaIpcMemHandle_t*>(handle64), ptr);
}
cudaError_t ztq_ipc_open(const void* handle64, void** ptr) {
    if (!ptr || !handle64) return cudaErrorInvalidValue;
    cudaIpcMemHandle_t h;
    memcpy(&h, handle64, sizeof(h));
    return cudaIpcOpenMemHandle(ptr, h, cudaIpcMemLazyEnablePeerAccess);
}
cudaError_t ztq_ipc_close(void* ptr) { return cudaIpcCloseMemHandle(ptr); }

size_t ztq_splitk_workspace_bytes(int N, int splits) {
    return (N > 0 && splits > 0) ? (size_t)N * splits * 4 : 0;
}

cudaError_t ztq_gemv_w4g_splitk(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                                int splits, void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream) {
    const int gs = group_shift(group);
    if (gs < 0 || K % group || !meta) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.w = static_cast<const uint8_t*>(qdata);
    p.meta = static_cast<const uint8_t*>(meta);
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = (K / group) * 4;
    p.gshift = gs;
    return gemv_splitk<F_W4G>(p, splits, group, workspace, workspace_bytes, flags, stream);
}

cudaError_t ztq_gemv_q4_0_splitk(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int splits,
                                 void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream) {
    if (!w_sep || K % 32 || data_offset < 0 || (data_offset & 15)) return cudaErrorInvalidValue;
    GemvParams p = {};
    p.meta = static_cast<const uint8_t*>(w_sep);
    p.w = p.meta + data_offset;
    p.x = x; p.y = y; p.N = N; p.K = K;
    p.row_bytes = K / 2;
    p.meta_row_bytes = K / 16;
    return gemv_splitk<F_Q4_0>(p, splits, 32, workspace, workspace_bytes, flags, stream);
}

// ---- split-K without a caller workspace ---------------------------------------
// Scratch for the fp32 partial sums lives in this file-scope device array: it is part of the library
// image, so every GPU that loads the library carries these bytes until the process exits.  In host code
// the array's name is only a handle for the runtime, not an address a kernel can use: the device address
// is looked up once per device with cudaGetSymbolAddress and that pointer is what the kernels receive.
static __device__ __align__(256) float g_splitk_static_scratch[ZTQ_STATIC_SCRATCH_BYTES / 4];

namespace {
constexpr int kMaxDevices = 64;
std::atomic<void*> g_scratch_ptr[kMaxDevices];

// Device address of the scratch array on the CURRENT device.  Only a successful lookup is remembered: a first
// call that fails (for instance because it was made while its stream was being captured, where the lookup is
// refused) leaves nothing behind, and the next call on that device tries again.
cudaError_t static_scratch(cudaStream_t stream, void** out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    void* p = g_scratch_ptr[dev].load(std::memory_order_acquire);
    if (!p) {
        cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(stream, &cs) == cudaSuccess && cs != cudaStreamCaptureStatusNone)
            return cudaErrorStreamCaptureUnsupported;      // the set-up call belongs before the capture
        e = cudaGetSymbolAddress(&p, g_splitk_static_scratch);
        if (e != cudaSuccess) return e;
        if (!p) return cudaErrorInvalidSymbol;
        g_scratch_ptr[dev].store(p, std::memory_order_release);   // every thread looks up the same address
    }
    *out = p;
    return cudaSuccess;
}
}  // namespace

cudaError_t ztq_gemv_w4g_splitk_static(const void* qdata, const void* meta, const void* x, void* y, int N, int K,
                                       int group, int splits, int flags, cudaStream_t stream) {
    if (N <= 0 || splits < 2) return cudaErrorInvalidValue;
    // the partial sums of this call must fit the built-in scratch: N * splits floats
    if ((size_t)N * (size_t)splits * sizeof(float) > (size_t)ZTQ_STATIC_SCRATCH_BYTES) return cudaErrorInvalidValue;
    void* scratch = nullptr;
    cudaError_t e = static_scratch(stream, &scratch);
    if (e != cudaSuccess) return e;
    return ztq_gemv_w4g_splitk(qdata, meta, x, y, N, K, group, splits, scratch, (size_t)ZTQ_STATIC_SCRATCH_BYTES, flags,
                               stream);
}

// K slices per row tile: cost model in steps of one group, a few steps of fixed cost per work item
static int tc_pick_slices(int n_tiles, int G, int sms) {
    int best = 1;
    long long best_cost = -1;
    for (int S = 1; S <= 8; ++S) {
        if (G % (4 * S)) continue;                            // slices of whole groups of four (scale loads, pairs)
        const long long waves = ceil_div((long long)n_tiles * S, sms);
        const long long cost = waves * (G / S + (S > 1 ? 14 : 6));          // a split item also pays fence, counter and the re-read
        if (best_cost < 0 || cost < best_cost) { best_cost = cost; best = S; }
    }
    return best;
}

struct TcLayout { int S; size_t counters_off, partial_off, total; };
static TcLayout tc_layout(int N, int K, int nbp, bool i8_sizes, int sms, int gb = 1) {
    TcLayout L;
    const int G = K / 128, n_tiles = ceil_div(N, 128);
    L.S = tc_pick_slices(n_tiles, G, sms);
    size_t off = (size_t)G * (tc_tile_bytes(nbp, i8_sizes) + tc_tail_bytes(nbp, i8_sizes, gb));
    off = (off + 255) & ~(size_t)255;
    L.counters_off = off;
    off += (size_t)n_tiles * 8 * 4;
    off = (off + 255) & ~(size_t)255;
    L.partial_off = off;
    if (L.S > 1) off += (size_t)L.S * nbp * N * 4;
    L.total = off;
    return L;
}

size_t ztq_gemm_w4g_tc_workspace_bytes(int N, int K, int batch) {
    if (N <= 0 || K <= 0 || batch <= 0) return 0;
    const int nbp = batch <= 16 ? 16 : 32;                  // sized for 16 columns even when 8 would do (the fp16 variant)
    return tc_layout(N, K, nbp, true, device_info().sms).total;       // the integer variant's tiles are the larger ones
}

static cudaError_t gemm_w4g_tc(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group, int batch,
                               void* workspace, size_t workspace_bytes, int flags, const ZtqAllReduce* ar, cudaStream_t stream) {
    if (!qdata || !meta || !x || !y || !workspace || N <= 0 || K <= 0 || batch <= 0) return cudaErrorInvalidValue;
    ArParams arp = {};
    const int pass = ar ? 16 : 32;                            // activation vectors per pass over the weights
    if (ar) {
        // integer operands only; every pass is one launch of the sequence all ranks count
        if ((flags & ZTQ_FP32_DECODE) || N > 65535 * 128) return cudaErrorInvalidValue;
        GemvParams gp = {};
        gp.N = N;
        cudaError_t e = fill_ar(gp, ar, batch < pass ? batch : pass);
        if (e != cudaSuccess) return e;
        arp = gp.ar;
    }
    // two groups per TMA box (K % 256), scales read eight groups at a time (16-byte aligned rows of meta: K % 512)
    if (group != 128 || K % 512 || (flags & (ZTQ_X_F32 | ZTQ_X_KB | ZTQ_Y_NB))) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(qdata) & 15) || (reinterpret_cast<uintptr_t>(x) & 15) ||
        (reinterpret_cast<uintptr_t>(meta) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 255))
        return cudaErrorInvalidValue;
    if (workspace_bytes < ztq_gemm_w4g_tc_workspace_bytes(N, K, batch)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return cudaErrorNotSupported;
    // the packed weights as a 2-D byte tensor [N rows][K/2 bytes]; boxes of 128 rows x 128 bytes, 128-byte swizzle
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)(K / 2), (cuuint64_t)N};
    const cuuint64_t strides[1] = {(cuuint64_t)(K / 2)};
    const cuuint32_t box[2] = {128, 128};
    const cuuint32_t estr[2] = {1, 1};
    if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(qdata), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    const bool pdl = !(flags & ZTQ_NO_PDL);
    const bool i8 = !(flags & ZTQ_FP32_DECODE);               // integer operands unless the caller forbids rounding x
    const int G = K / 128;
    const int tiles = ceil_div(N, 128);
    const size_t ye = (flags & ZTQ_Y_F32) ? 4 : 2;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    for (int b0 = 0; b0 < batch; b0 += pass) {
        const int nb = batch - b0 < pass ? batch - b0 : pass;
        const int nbp = (nb <= 8 && i8) ? 8 : nb <= 16 ? 16 : 32;     // an MMA's cost grows with its N: 32 / 48 / 96 columns
        const TcLayout L = tc_layout(N, K, nbp, true, dev.sms);        // offsets sized for the larger (integer) tiles
        unsigned* counters = reinterpret_cast<unsigned*>(ws + L.counters_off);
        const __half* xb = static_cast<const __half*>(x) + (size_t)b0 * K;
        cudaError_t e = i8 ? launch(tc_prepare_x_i8_kernel, dim3(G), dim3(8 * nbp), 0, stream, pdl, xb, ws, K, nb, nbp,
                                    counters, tiles * 8)
                           : launch(tc_prepare_x_kernel, dim3(G), dim3(256), 0, stream, pdl, xb, ws, K, nb, nbp, counters,
                                    tiles * 8);
        if (e != cudaSuccess) return e;
        TcParams tp = {};
        tp.meta = static_cast<const uint32_t*>(meta);
        tp.xprep = ws;
        tp.y = static_cast<uint8_t*>(y) + (size_t)b0 * N * ye;
        tp.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
        tp.N = N; tp.K = K; tp.batch = nb; tp.G = G;
        tp.nmma = nbp;
        tp.S = L.S;
        tp.Gs = G / L.S;
        tp.partial = L.S > 1 ? reinterpret_cast<float*>(ws + L.partial_off) : nullptr;
        tp.counters = counters;
        tp.ar = arp;
        const int items = tiles * L.S;
        const int grid = items < dev.sms ? items : dev.sms;
        if (ar && ceil_div(items, grid) > kTcArPend) return cudaErrorInvalidValue;     // more tiles per CTA than its list of pending tiles holds
        const int tile_bytes = tc_tile_bytes(nbp, i8);
        const size_t smem = (size_t)kTcStages * kTcRawBytes + (size_t)tc_bring(tile_bytes) * tile_bytes +
                            (size_t)kTcTailSlots * kTcTailGroups * tc_tail_bytes(nbp, i8) + 96 * 8 + 64 + (ar ? kTcArSmem : 0);
        const bool split = L.S > 1;
        if (ar && nbp == 8) e = split ? launch_tc<8, true, true, 1, true>(map, tp, grid, smem, stream, pdl) : launch_tc<8, true, false, 1, true>(map, tp, grid, smem, stream, pdl);
        else if (ar) e = split ? launch_tc<16, true, true, 1, true>(map, tp, grid, smem, stream, pdl) : launch_tc<16, true, false, 1, true>(map, tp, grid, smem, stream, pdl);
        else if (i8 && nbp == 8) e = split ? launch_tc<8, true, true>(map, tp, grid, smem, stream, pdl) : launch_tc<8, true, false>(map, tp, grid, smem, stream, pdl);
        else if (i8 && !split) e = nbp == 16 ? launch_tc<16, true, false>(map, tp, grid, smem, stream, pdl) : launch_tc<32, true, false>(map, tp, grid, smem, stream, pdl);
        else if (i8) e = nbp == 16 ? launch_tc<16, true, true>(map, tp, grid, smem, stream, pdl) : launch_tc<32, true, true>(map, tp, grid, smem, stream, pdl);
        else if (!split) e = nbp == 16 ? launch_tc<16, false, false>(map, tp, grid, smem, stream, pdl) : launch_tc<32, false, false>(map, tp, grid, smem, stream, pdl);
        else e = nbp == 16 ? launch_tc<16, false, true>(map, tp, grid, smem, stream, pdl) : launch_tc<32, false, true>(map, tp, grid, smem, stream, pdl);
        if (e != cudaSuccess) return e;
    }
    return cudaGetLastError();
}

cudaError_t ztq_gemm_w4g_tc(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group, int batch,
                            void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream) {
    return gemm_w4g_tc(qdata, meta, x, y, N, K, group, batch, workspace, workspace_bytes, flags, nullptr, stream);
}

cudaError_t ztq_gemm_w4g_tc_allreduce(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                                      int batch, void* workspace, size_t workspace_bytes, int flags, const ZtqAllReduce* ar,
                                      cudaStream_t stream) {
    if (!ar) return cudaErrorInvalidValue;
    return gemm_w4g_tc(qdata, meta, x, y, N, K, group, batch, workspace, workspace_bytes, flags, ar, stream);
}

// ---- launch plan of a shape, for tests and tools ------------------------------------
// Which kernel a call with these arguments launches first, and the tiling it uses.  `sms` stands in for the SM
// count (so the answer can be had without a device).  fmt: 0 Q4_0, 1 IQ4_NL, 2 W4G, 3 Q8_0, 4 ternary, 5 Q4_K,
// 6 Q5_K, 7 Q6_K, 8 W4G on the tensor cores.  out[0..11] =
//   GEMV:   {kernel (0 plain, 1 streaming, 2 chunk-pair), batch columns per launch, RT, R, S, Sx, P, grid,
//            tiles of the busiest CTA, passes of the busiest CTA, WPT, teams}
//   tensor: {3, padded columns, K slices, groups per slice, row tiles, work items, grid, items of the busiest CTA,
//            0, 0, 0, 0}
// Returns 0, or 1 when the arguments are not a valid problem.
int ztq_describe_plan(int fmt, int N, int K, int group, int batch, int sms, int* out) {
    if (!out || N <= 0 || K <= 0 || batch <= 0 || sms <= 0) return 1;
    for (int i = 0; i < 12; ++i) out[i] = 0;
    DeviceInfo dev;
    dev.sms = sms;
    dev.major = 10;
    if (fmt == 8) {
        if (group != 128 || K % 512) return 1;
        const int nb = batch < 32 ? batch : 32;
        const int nbp = nb <= 8 ? 8 : nb <= 16 ? 16 : 32;
        const TcLayout L = tc_layout(N, K, nbp, true, sms);
        const int tiles = ceil_div(N, 128), items = tiles * L.S, grid = items < sms ? items : sms;
        const int v[8] = {3, nbp, L.S, (K / 128) / L.S, tiles, items, grid, ceil_div(items, grid)};
        for (int i = 0; i < 8; ++i) out[i] = v[i];
        return 0;
    }
    GemvParams p = {};
    p.w = reinterpret_cast<const uint8_t*>(uintptr_t(256));       // aligned stand-ins: only their alignment is looked at
    p.meta = p.w;
    p.N = N; p.K = K;
    p.xs_b = K; p.xs_k = 1; p.ys_b = N; p.ys_n = 1;
    Plan pl1, pl2, plp;
    auto fill = [&](const Plan& pl, int kernel, int bc) {
        const int rows = ceil_div(N, pl.grid), tiles = ceil_div(rows, pl.p.R);
        const int v[12] = {kernel, bc, pl.rt, pl.p.R, pl.p.S, pl.p.Sx, pl.p.P, pl.grid, tiles,
                           ceil_div(tiles, pl.p.P / pl.p.R), pl.p.WPT, pl.p.T};
        for (int i = 0; i < 12; ++i) out[i] = v[i];
    };
    switch (fmt) {
        case F_Q4_0: case F_IQ4NL:
            if (K % 32) return 1;
            p.row_bytes = K / 2; p.meta_row_bytes = K / 16;
            break;
        case F_W4G: {
            const int gs = group_shift(group);
            if (gs < 0 || K % group) return 1;
            p.row_bytes = K / 2; p.meta_row_bytes = (K / group) * 4; p.gshift = gs;
            break;
        }
        case F_Q8_0:
            if (K % 32) return 1;
            p.row_bytes = (K / 32) * 36;
            break;
        case F_TERN:
            if (K % 64) return 1;
            p.row_bytes = K / 4;
            break;
        case F_Q4K: case F_Q5K: case F_Q6K:
            if (K % 256) return 1;
            p.row_bytes = K / 2;
            p.meta_row_bytes = K / 256 * (fmt == F_Q6K ? 96 : fmt == F_Q5K ? 48 : 16);
            break;
        default:
            return 1;
    }
    switch (fmt) {
        case F_Q4_0: pl2 = make_plan<F_Q4_0>(p, 2, dev); pl1 = make_plan<F_Q4_0>(p, 1, dev); plp = make_pair_plan<F_Q4_0>(p, dev); break;
        case F_IQ4NL: pl2 = make_plan<F_IQ4NL>(p, 2, dev); pl1 = make_plan<F_IQ4NL>(p, 1, dev); break;
        case F_W4G: pl2 = make_plan<F_W4G>(p, 2, dev); pl1 = make_plan<F_W4G>(p, 1, dev);
                    if (p.gshift == 2) plp = make_pair_plan<F_W4G>(p, dev); break;
        case F_Q8_0: pl2 = make_plan<F_Q8_0>(p, 2, dev); pl1 = make_plan<F_Q8_0>(p, 1, dev); break;
        case F_TERN: pl1 = make_plan<F_TERN>(p, 1, dev); break;
        case F_Q4K: plp = make_pair_plan<F_Q4K>(p, dev); break;
        case F_Q5K: plp = make_pair_plan<F_Q5K>(p, dev); break;
        default: plp = make_pair_plan<F_Q6K>(p, dev); break;
    }
    if (fmt >= F_Q4K) {
        if (!plp.ok) return 1;
        fill(plp, 2, 1);
        return 0;
    }
    if (!pl1.ok) { out[0] = 0; out[1] = batch; return 0; }        // the plain kernel: one warp per row
    const bool two = batch >= 2 && pl2.ok && pl2.spt == 1;
    if (two) fill(pl2, 1, 2);
    else if (plp.ok && (long long)N >= 12LL * sms) fill(plp, 2, 1);
    else fill(pl1, 1, 1);
    return 0;
}

// ---- Q4_0 with three or more activation rows: the same tensor-core kernel, a scale per block of 32 ----------
size_t ztq_gemm_q4_0_tc_workspace_bytes(int N, int K, int batch) {
    if (N <= 0 || K <= 0 || batch <= 0) return 0;
    return tc_layout(N, K, 16, true, device_info().sms, 4).total;                   // sized for 16 columns per pass
}

cudaError_t ztq_gemm_q4_0_tc(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch, void* workspace,
                             size_t workspace_bytes, int flags, cudaStream_t stream) {
    if (!w_sep || !x || !y || !workspace || N <= 0 || K <= 0 || batch <= 0 || data_offset <= 0 || (data_offset & 15)) return cudaErrorInvalidValue;
    if (K % 512 || (flags & ~(ZTQ_Y_F32 | ZTQ_NO_PDL))) return cudaErrorInvalidValue;
    const uint8_t* qdata = static_cast<const uint8_t*>(w_sep) + data_offset;
    if ((reinterpret_cast<uintptr_t>(w_sep) & 15) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 255))
        return cudaErrorInvalidValue;
    if (workspace_bytes < ztq_gemm_q4_0_tc_workspace_bytes(N, K, batch)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return cudaErrorNotSupported;
    CUtensorMap map;                                           // the data region as [N rows][K/2 bytes], like the W4A16 codes
    const cuuint64_t dims[2] = {(cuuint64_t)(K / 2), (cuuint64_t)N};
    const cuuint64_t strides[1] = {(cuuint64_t)(K / 2)};
    const cuuint32_t box[2] = {128, 128};
    const cuuint32_t estr[2] = {1, 1};
    if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(qdata), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    const bool pdl = !(flags & ZTQ_NO_PDL);
    const int G = K / 128, tiles = ceil_div(N, 128);
    const size_t ye = (flags & ZTQ_Y_F32) ? 4 : 2;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    for (int b0 = 0; b0 < batch; b0 += 16) {                   // 16 activation vectors per pass over the weights
        const int nb = batch - b0 < 16 ? batch - b0 : 16;
        const int nbp = nb <= 8 ? 8 : 16;
        const TcLayout L = tc_layout(N, K, nbp, true, dev.sms, 4);
        unsigned* counters = reinterpret_cast<unsigned*>(ws + L.counters_off);
        const __half* xb = static_cast<const __half*>(x) + (size_t)b0 * K;
        cudaError_t e = launch(tc_prepare_x_i8_q4_0_kernel, dim3(G), dim3(8 * nbp), 0, stream, pdl, xb, ws, K, nb, nbp, counters, tiles * 8);
        if (e != cudaSuccess) return e;
        TcParams tp = {};
        tp.meta = static_cast<const uint32_t*>(w_sep);         // fp16 scales, one per block of 32, rows of K / 32
        tp.xprep = ws;
        tp.y = static_cast<uint8_t*>(y) + (size_t)b0 * N * ye;
        tp.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
        tp.N = N; tp.K = K; tp.batch = nb; tp.G = G;
        tp.nmma = nbp;
        tp.S = L.S;
        tp.Gs = G / L.S;
        tp.partial = L.S > 1 ? reinterpret_cast<float*>(ws + L.partial_off) : nullptr;
        tp.counters = counters;
        const int items = tiles * L.S;
        const int grid = items < dev.sms ? items : dev.sms;
        const int tile_bytes = tc_tile_bytes(nbp, true);
        const size_t smem = (size_t)kTcStages * kTcRawBytes + (size_t)tc_bring(tile_bytes) * tile_bytes +
                            (size_t)kTcTailSlots * kTcTailGroups * tc_tail_bytes(nbp, true, 4) + 96 * 8 + 64;
        const bool split = L.S > 1;
        if (nbp == 8) e = split ? launch_tc<8, true, true, 4>(map, tp, grid, smem, stream, pdl) : launch_tc<8, true, false, 4>(map, tp, grid, smem, stream, pdl);
        else e = split ? launch_tc<16, true, true, 4>(map, tp, grid, smem, stream, pdl) : launch_tc<16, true, false, 4>(map, tp, grid, smem, stream, pdl);
        if (e != cudaSuccess) return e;
    }
    return cudaGetLastError();
}

// ---- Q8_0 with three or more activation rows: the same kernel on the raw 36-byte blocks ---------------------------
size_t ztq_gemm_q8_0_tc_workspace_bytes(int N, int K, int batch) {
    if (N <= 0 || K <= 0 || batch <= 0) return 0;
    return tc_layout(N, K, 16, true, device_info().sms, 4).total;
}

cudaError_t ztq_gemm_q8_0_tc(const void* blocks36, const void* x, void* y, int N, int K, int batch, void* workspace,
                             size_t workspace_bytes, int flags, cudaStream_t stream) {
    if (!blocks36 || !x || !y || !workspace || N <= 0 || K <= 0 || batch <= 0) return cudaErrorInvalidValue;
    if (K % 512 || (flags & ~(ZTQ_Y_F32 | ZTQ_NO_PDL))) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(blocks36) & 15) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 255))
        return cudaErrorInvalidValue;
    if (workspace_bytes < ztq_gemm_q8_0_tc_workspace_bytes(N, K, batch)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return cudaErrorNotSupported;
    // the blocks of a row as bytes: [N rows][K / 32 * 36 bytes]; one box = the four blocks of a group x 128 rows
    CUtensorMap map;
    const cuuint64_t row_bytes = (cuuint64_t)(K / 32) * 36;     // a multiple of 16: K % 512 == 0
    const cuuint64_t dims[2] = {row_bytes, (cuuint64_t)N};
    const cuuint64_t strides[1] = {row_bytes};
    const cuuint32_t box[2] = {144, 128};
    const cuuint32_t estr[2] = {1, 1};
    if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(blocks36), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    const bool pdl = !(flags & ZTQ_NO_PDL);
    const int G = K / 128, tiles = ceil_div(N, 128);
    const size_t ye = (flags & ZTQ_Y_F32) ? 4 : 2;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    for (int b0 = 0; b0 < batch; b0 += 16) {                   // 16 activation vectors per pass over the weights
        const int nb = batch - b0 < 16 ? batch - b0 : 16;
        const int nbp = nb <= 8 ? 8 : 16;
        const TcLayout L = tc_layout(N, K, nbp, true, dev.sms, 4);
        unsigned* counters = reinterpret_cast<unsigned*>(ws + L.counters_off);
        const __half* xb = static_cast<const __half*>(x) + (size_t)b0 * K;
        cudaError_t e = launch(tc_prepare_x_i8_q8_0_kernel, dim3(G), dim3(8 * nbp), 0, stream, pdl, xb, ws, K, nb, nbp, counters, tiles * 8);
        if (e != cudaSuccess) return e;
        TcParams tp = {};
        tp.meta = nullptr;                                     // the scales travel with the blocks
        tp.xprep = ws;
        tp.y = static_cast<uint8_t*>(y) + (size_t)b0 * N * ye;
        tp.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
        tp.N = N; tp.K = K; tp.batch = nb; tp.G = G;
        tp.nmma = nbp;
        tp.S = L.S;
        tp.Gs = G / L.S;
        tp.partial = L.S > 1 ? reinterpret_cast<float*>(ws + L.partial_off) : nullptr;
        tp.counters = counters;
        const int items = tiles * L.S;
        const int grid = items < dev.sms ? items : dev.sms;
        const int tile_bytes = tc_tile_bytes(nbp, true);
        const size_t smem = (size_t)kTcStagesW8 * kTcRawBytesW8 + (size_t)kTcBRingW8 * tile_bytes +
                            (size_t)kTcTailSlots * kTcTailGroups * tc_tail_bytes(nbp, true, 4) + kTcScaleBytes + 96 * 8 + 64;
        const bool split = L.S > 1;
        if (nbp == 8) e = split ? launch_tc<8, true, true, 4, false, true>(map, tp, grid, smem, stream, pdl) : launch_tc<8, true, false, 4, false, true>(map, tp, grid, smem, stream, pdl);
        else e = split ? launch_tc<16, true, true, 4, false, true>(map, tp, grid, smem, stream, pdl) : launch_tc<16, true, false, 4, false, true>(map, tp, grid, smem, stream, pdl);
        if (e != cudaSuccess) return e;
    }
    return cudaGetLastError();
}

// ---- reference-named launchers -------------------------------------------
// gemm_q4_f32 / gemm_q8_f32: C[M,N] = A[M,K] * B[K,N] with the weights as A, so
// the activations arrive as [K, batch] and the result leaves as [M, batch].
cudaError_t gemm_q4_f32(const void* A_q4, const float* B, float* C, int M, int K, int N, int data_offset,
                        cudaStream_t stream) {
    if (K % 32 != 0) return cudaErrorInvalidValue;             // same check as gemm_q4.cu:169-171
    return ztq_gemv_q4_0(A_q4, data_offset, B, C, M, K, N, ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_X_KB | ZTQ_Y_NB, stream);
}

cudaError_t gemm_q8_f32(const void* A_q8, const float* B, float* C, int M, int K, int N, cudaStream_t stream) {
    if (K % 32 != 0) return cudaErrorInvalidValue;
    return ztq_gemv_q8_0(A_q8, B, C, M, K, N, ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_X_KB | ZTQ_Y_NB, stream);
}

// Any K: rows that are not a multiple of 64 codes take the per-element kernel.
namespace ztq {
__global__ void ternary_rows_any_kernel(const uint8_t* __restrict__ w, const float* __restrict__ x,
                                        float* __restrict__ y, int M, int K) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= M) return;
    const int rb = (K + 3) / 4;
    const uint8_t* wr = w + (size_t)row * rb;
    float acc = 0.f;
    for (int c = lane; c < rb; c += 32) {
        const uint32_t byte = wr[c];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int k = c * 4 + t;
            if (k < K) {
                const uint32_t code = (byte >> (2 * t)) & 3u;
                if (code == 2u) acc += x[k];
                else if (code == 0u) acc -= x[k];
            }
        }
    }
    acc = warp_sum(acc);
    if (lane == 0) y[row] = acc;
}
}  // namespace ztq

cudaError_t ternary_gemv_f32(const void* W_ternary, const float* x, float* y, int M, int K, cudaStream_t stream) {
    if (!W_ternary || !x || !y || M <= 0 || K <= 0) return cudaErrorInvalidValue;
    if (K % 64 == 0)
        return ztq_gemv_ternary(W_ternary, nullptr, x, y, M, K, 1, ZTQ_X_F32 | ZTQ_Y_F32, stream);
    cudaError_t e = launch(ztq::ternary_rows_any_kernel, dim3(ceil_div(M, 8)), dim3(256), 0, stream, true,
                           static_cast<const uint8_t*>(W_ternary), x, y, M, K);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// ---- residency helpers -------------------------------------------------------
cudaError_t ztq_repack_blocks18(const void* aos, void* sep, long long n_blocks, cudaStream_t stream) {
    if (!aos || !sep || n_blocks <= 0) return cudaErrorInvalidValue;
    const long long data_off = (n_blocks * 2 + 15) & ~15LL;
    const long long threads = n_blocks * 9;
    repack_blocks18_kernel<<<ceil_div(threads, 256), 256, 0, stream>>>(static_cast<const uint8_t*>(aos),
                                                                       static_cast<uint8_t*>(sep), n_blocks, data_off);
    return cudaGetLastError();
}

cudaError_t ztq_pack_w4g_meta(const void* scales, const void* zeros, void* meta, long long n_groups,
                              cudaStream_t stream) {
    if (!scales || !zeros || !meta || n_groups <= 0) return cudaErrorInvalidValue;
    pack_w4g_meta_kernel<<<ceil_div(n_groups, 256), 256, 0, stream>>>(static_cast<const uint16_t*>(scales),
                                                                      static_cast<const uint16_t*>(zeros),
                                                                      static_cast<uint32_t*>(meta), n_groups);
    return cudaGetLastError();
}

cudaError_t ztq_repack_ternary_rows(const void* flat, void* rows, int M, int K, cudaStream_t stream) {
    if (!flat || !rows || M <= 0 || K <= 0) return cudaErrorInvalidValue;
    const long long total = (long long)M * ((K + 3) / 4);
    repack_ternary_rows_kernel<<<ceil_div(total, 256), 256, 0, stream>>>(static_cast<const uint8_t*>(flat),
                                                                         static_cast<uint8_t*>(rows), M, K);
    return cudaGetLastError();
}

cudaError_t ztq_quantize_q4_0(const float* src, void* sep, long long n, cudaStream_t stream) {
    if (!src || !sep || n <= 0 || n % 32) return cudaErrorInvalidValue;
    const long long nb = n / 32;
    const long long data_off = (nb * 2 + 15) & ~15LL;
    quantize_block32_kernel<4><<<ceil_div(nb * 8, 256), 256, 0, stream>>>(src, static_cast<uint8_t*>(sep), nb, data_off);
    return cudaGetLastError();
}

cudaError_t ztq_quantize_q8_0(const float* src, void* blocks36, long long n, cudaStream_t stream) {
    if (!src || !blocks36 || n <= 0 || n % 32) return cudaErrorInvalidValue;
    const long long nb = n / 32;
    quantize_block32_kernel<8><<<ceil_div(nb * 8, 256), 256, 0, stream>>>(src, static_cast<uint8_t*>(blocks36), nb, 0);
    return cudaGetLastError();
}

cudaError_t ztq_quantize_w4g(const float* src, void* qdata, void* meta, long long n, int group, int awq_rounding,
                             cudaStream_t stream) {
    if (!src || !qdata || !meta || n <= 0 || group <= 0 || group % 2 || n % group) return cudaErrorInvalidValue;
    const long long ng = n / group;
    if (group == 128)
        quantize_w4g128_kernel<<<ceil_div(ng * 32, 256), 256, 0, stream>>>(src, static_cast<uint8_t*>(qdata),
                                                                           static_cast<uint32_t*>(meta), ng, awq_rounding);
    else
        quantize_w4g_generic_kernel<<<ceil_div(ng, 128), 128, 0, stream>>>(src, static_cast<uint8_t*>(qdata),
                                                                           static_cast<uint32_t*>(meta), ng, group, awq_rounding);
    return cudaGetLastError();
}

cudaError_t ztq_dequantize(int fmt, const void* w, const void* meta_or_null, float* dst, long long n, int aux,
                           cudaStream_t stream) {
    if (!w || !dst || n <= 0 || fmt < 0 || fmt > 4) return cudaErrorInvalidValue;
    const uint8_t* wp = static_cast<const uint8_t*>(w);
    const uint8_t* mp = static_cast<const uint8_t*>(meta_or_null);
    if (fmt == F_Q4_0 || fmt == F_IQ4NL) {       // separated buffer: scales first, data at byte `aux`
        if (aux < 0 || n % 32) return cudaErrorInvalidValue;
        mp = wp;
        wp = wp + aux;
    } else if (fmt == F_W4G) {
        if (!mp || aux <= 0 || n % aux) return cudaErrorInvalidValue;
    } else if (fmt == F_TERN) {
        if (aux <= 0 || n % aux) return cudaErrorInvalidValue;
    } else if (n % 32) {
        return cudaErrorInvalidValue;
    }
    dequantize_kernel<<<ceil_div(n, 256), 256, 0, stream>>>(fmt, wp, mp, dst, n, aux);
    return cudaGetLastError();
}

cudaError_t ztq_matmul_wkn_f32(const void* x, const float* w_kn, float* y, int M, int K, int N, int flags, cudaStream_t stream) {
    if (!x || !w_kn || !y || M <= 0 || K <= 0 || N <= 0 || (flags & ~(ZTQ_X_F32 | ZTQ_NO_PDL))) return cudaErrorInvalidValue;
    const long long total = (long long)M * N;
    cudaError_t e = launch(matmul_wkn_kernel, dim3(ceil_div(total, 256)), dim3(256), 0, stream, !(flags & ZTQ_NO_PDL), x, w_kn, y, M, K, N,
                           (flags & ZTQ_X_F32) ? 1 : 0);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// ---- probes ------------------------------------------------------------------
namespace ztq {
// A kernel with the launch shape of a GEMV and no work: what a dependent launch costs before any byte moves.
__global__ void launch_floor_kernel(int* sink) {
    extern __shared__ __align__(128) uint8_t floor_smem[];
    grid_dep_launch();
    grid_dep_wait();
    if (sink && threadIdx.x == 0 && blockIdx.x == 0x7fffffff) *sink = floor_smem[0];
}
}  // namespace ztq

cudaError_t ztq_probe_launch(int grid, int threads, int smem_bytes, int flags, cudaStream_t stream) {
    if (grid <= 0 || threads <= 0 || threads > 1024 || smem_bytes < 0 || smem_bytes > 227 * 1024) return cudaErrorInvalidValue;
    static std::atomic<unsigned> done_mask{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned bit = 1u << (dev & 31);
    if (!(done_mask.load(std::memory_order_acquire) & bit)) {
        cudaError_t e = cudaFuncSetAttribute(ztq::launch_floor_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        done_mask.fetch_or(bit, std::memory_order_release);
    }
    cudaError_t e = launch(ztq::launch_floor_kernel, dim3(grid), dim3(threads), (size_t)smem_bytes, stream, !(flags & ZTQ_NO_PDL),
                           static_cast<int*>(nullptr));
    return e != cudaSuccess ? e : cudaGetLastError();
}

int ztq_check_sm100(void) { return device_info().major == 10 ? 1 : 0; }

int ztq_abi_version(void) { return 1; }

int ztq_device_error(void) {
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    int first = 0;
    for (auto take : {&take_error, &ztq_take_error_step, &ztq_take_error_attn}) {  // one word per translation unit: all are cleared
        const int e = take();
        if (first == 0) first = e;
    }
    return first;
}

}  // extern "C"
