// attn_tc.cuh -- the attention of attn_q8.cuh for sequences with many new tokens (prompts), on the tcgen05 tensor cores.
//
// An item is (sequence, 256 rows, kv head) and one CTA; its rows are two tiles of 128 (M of the products).  Per step of 128
// keys:
//   S_t = Q_t K^T   (fp16 x fp16 -> fp32 in TMEM, 128 columns)            Q_t, K from shared memory
//   P_t = 2^(S_t f - c + lift) sv as fp16, over the columns of S_t
//   O_t += P_t V    (P_t from TMEM, V^T from shared memory; D columns)
// The codes become fp16 operands (exactly) on the way into shared memory, once per step for both tiles: a step's 64 KB of
// operands cost what a quarter of the exponentials costs.  The scales stay out of the operands: sixteen keys are a chunk of
// scores in the softmax, whose exponent's factor takes sk and whose weights take sv.
//
// Roles of the warps: 0-3 and 4-7 softmax of tile 0 and 1 (a thread is a row: TMEM lane), then kTcaConv for K codes ->
// operand and kTcaConv for V (loaded one step ahead, their blocks and scales two), the last issues the products.  The two
// tiles alternate: while one is in its softmax the tensor cores work for the other.  The reference c of a row
// (attn_q8.cuh) moves only when exceeded by more than a slack; then the row's O is rescaled in TMEM.
// Operands stand in the canonical K-major layout without swizzle: core matrices of 8 rows x 16 bytes, 128 bytes apart along
// the contraction; both store patterns below are free of bank conflicts.
//
// What bounds it: per step and SM there are 2048 clocks of tensor time, the same of exponentials (16 per clock) and the same of
// shared-memory traffic, but the chain scores -> maximum -> weights -> products of two tiles overlaps them only in part: 4096
// new tokens over 8192 keys, 32 / 8 heads of 128 take 590 us (700 TFLOP/s), the products alone 325, without the conversions
// 434, without the exponentials 481.  P is rounded to fp16 like the outputs, whose error against 64 bits that raises from 2.1e-4 to
// 2.9e-4 of their norm.  96 registers per thread (17 warps) spill 66 to 132 bytes.
//
// With fp32 inputs or outputs (SPLIT) an item is one tile of 128 rows: its queries are two fp16 terms (of the row times a power of two,
// which its scores are divided by) in the places of the two tiles, its weights two terms with the second in the columns of the second tile's scores, and every product is done for both.
//
// With few items the keys are cut into `splits` ranges of steps; a CTA then leaves {max, sum, rows} in the workspace and
// attn_tc_join_kernel adds the ranges in order.
#pragma once

#include "attn_q8.cuh"
#include "tc_common.cuh"

#include <type_traits>

namespace ztq {

constexpr int kTcaKeys = 128;
__host__ __device__ constexpr int tca_rows(bool split) { return split ? 128 : 256; }     // rows of an item
constexpr int kTcaConv = 4;                      // warps that convert K, and as many V (two each leave 128 registers per thread: 596 against 589 us)
constexpr int kTcaGroups = 8 / kTcaConv;         // groups of 16 keys that each of them takes
constexpr int kTcaMma = 8 + 2 * kTcaConv;
constexpr int kTcaThreads = 32 * (kTcaMma + 1);

struct __align__(16) TcaInfo {                  // one step's factors, by groups of 16 keys
    float ks[8], vs[8], ve[8];                  // |K scale|; V scale, 0 where it is not finite; its exponent
    uint32_t hidden, bad_v;                     // groups without a block; groups whose V scale is not finite
};

struct TcaShared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], info_full[4];
    TcaInfo info[4];
    uint32_t tmem;
    float down[128];                            // fp32 queries: what a row's scores are multiplied by
};
static_assert(sizeof(TcaShared) <= 2048, "the end of tca_smem");
template <int D>
__host__ __device__ constexpr int tca_smem() {
    const int n = 256 * D * 2 + 4 * kTcaKeys * D * 2 + 2048;
    return n < 120 * 1024 ? 120 * 1024 : n;     // one CTA per SM: it holds all of TMEM
}

struct TcaParams {
    AttnParams a;
    int splits, rows;                           // rows of an item
    float* parts;                               // [item][split][rows][D + 2]
};

struct TcaItem {
    int b, r0, r1, h, lo, hi;
    AttnSeq s;
};
// upto[b]: items of sequences 0 .. b for one kv head
__device__ __forceinline__ void tca_scan(const AttnParams& p, int tile, int* upto, int* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int before = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int v = b < p.seqs ? (attn_seq(p, b).rows(p.group) + tile - 1) / tile : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        __syncthreads();
        if (lane == 31) part[warp] = v;
        __syncthreads();
        int all = before;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) v += part[w];
            all += part[w];
        }
        if (b < p.seqs) upto[b] = before + v;
        before = all;
    }
    __syncthreads();
}
// Item i, or false behind the last.  Within a sequence the items with most keys come first: the hardware deals CTAs in
// order, so the short ones fill the end.
__device__ __forceinline__ bool tca_item(const AttnParams& p, int tile, const int* upto, long long i, TcaItem& it) {
    const int pair = (int)(i / p.kv_heads);
    it.h = (int)(i % p.kv_heads);
    if (pair >= upto[p.seqs - 1]) return false;
    int lo = 0, hi = p.seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] > pair) hi = mid; else lo = mid + 1;
    }
    it.b = lo;
    it.s = attn_seq(p, lo);
    const int rows = it.s.rows(p.group);
    it.r0 = (upto[lo] - 1 - pair) * tile;
    it.r1 = min(it.r0 + tile, rows);
    attn_span(p, it.s, it.r0, it.r1, it.lo, it.hi);
    return true;
}

__device__ __forceinline__ void tc_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// Sixteen columns, not waited for; tc_wait16 names the registers, so nothing that uses them moves in front of it.
__device__ __forceinline__ void tc_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tc_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t turned(uint32_t x, bool plus) { return plus ? unbias(x) : unbias(x) ^ 0x80008000u; }

template <int D, bool SPLIT>
__global__ void __launch_bounds__(kTcaThreads, 1) attn_tc_kernel(const TcaParams tp) {
    constexpr int CG = D / 8;                               // 16-byte columns of a K-major row of D
    constexpr int QB = 128 * D * 2, KB = kTcaKeys * D * 2;  // bytes of a tile of Q, of a K or V operand
    constexpr uint32_t kS = 0, kO = 256;                    // TMEM columns of the score tiles and of the outputs
    extern __shared__ __align__(1024) uint8_t smem_tc[];
    uint8_t* sq = smem_tc;
    uint8_t* sk = smem_tc + 2 * QB;
    uint8_t* sv = sk + 2 * KB;
    TcaShared& sh = *reinterpret_cast<TcaShared*>(sv + 2 * KB);
    const AttnParams& p = tp.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    grid_dep_wait();
    // the scan's scratch lies where the operands will be
    int* upto = reinterpret_cast<int*>(sk);
    tca_scan(p, tca_rows(SPLIT), upto, reinterpret_cast<int*>(sv));
    TcaItem it;
    const bool mine = tca_item(p, tca_rows(SPLIT), upto, blockIdx.x, it);
    __syncthreads();
    if (!mine) return;
    const int kt_lo = it.lo / kTcaKeys, kt_all = max(0, (it.hi + kTcaKeys - 1) / kTcaKeys - kt_lo);
    const int kt0 = kt_lo + (int)((long long)kt_all * blockIdx.y / tp.splits), kt1 = kt_lo + (int)((long long)kt_all * (blockIdx.y + 1) / tp.splits);
    const int n = kt1 - kt0, rows = it.r1 - it.r0, tiles = !SPLIT && rows > 128 ? 2 : 1;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], kTcaConv); mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], kTcaConv); mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.s_full[i], 1); mbar_init(&sh.p_full[i], 128); mbar_init(&sh.o_full[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sh.info_full[i], 2);
        mbar_fence_init();
    }
    if (warp == kTcaMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        // only now: a kernel behind this one that takes tensor memory before its own wait would otherwise wait for this one's end while
        // holding what this CTA has yet to get
        grid_dep_launch();
    }
    // queries: 16-byte pieces in K-major order, a phase of eight lanes writes eight rows of one column; scores use |scale|
    auto query_at = [&](int row) { return (it.s.first + row / p.group) * p.q_token + (long long)(it.h * p.group + row % p.group) * p.q_head; };
    auto place = [&](int r, int col) { return sq + (r >> 3) * (CG * 128) + col * 128 + (r & 7) * 16; };
    if (SPLIT && p.x_f32) {
        // a warp takes eight rows: a lane a row's columns lane / 8 + 4 j
        for (int r = 8 * warp + (lane & 7); r < 128; r += kTcaThreads / 4) {
            const int row = it.r0 + r;
            float x[CG / 4][8], top = 0.f;
#pragma unroll
            for (int j = 0; j < CG / 4; ++j) {
                const float* src = static_cast<const float*>(p.q) + query_at(row) + 8 * (4 * j + (lane >> 3));
                if (row >= it.r1) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[j][k] = 0.f;
                } else if (p.vec) {
                    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
                    x[j][0] = a.x; x[j][1] = a.y; x[j][2] = a.z; x[j][3] = a.w;
                    x[j][4] = b.x; x[j][5] = b.y; x[j][6] = b.z; x[j][7] = b.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[j][k] = src[k];
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[j][k]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            float up = attn_up(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)));
            if (lane < 8) sh.down[r] = attn_down(up);
            if (p.scale_log2 < 0) up = -up;
#pragma unroll
            for (int j = 0; j < CG / 4; ++j) {
                uint32_t v[4], rest[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float a = x[j][2 * k] * up, b = x[j][2 * k + 1] * up;
                    v[k] = pack_half2(a, b);
                    rest[k] = pack_rest(a, b, v[k]);
                }
                uint8_t* dst = place(r, 4 * j + (lane >> 3));
                *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<uint4*>(dst + QB) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            }
        }
    } else {
        for (int i = tid; i < tiles * 128 * CG; i += kTcaThreads) {
            const int r = (i & 7) + (i >> 3) / CG * 8, col = (i >> 3) % CG, row = it.r0 + r;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < it.r1) {
                const __half* src = static_cast<const __half*>(p.q) + query_at(row) + 8 * col;
                if (p.vec) {
                    const uint2 a = *reinterpret_cast<const uint2*>(src), b = *reinterpret_cast<const uint2*>(src + 4);
                    v = make_uint4(a.x, a.y, b.x, b.y);
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)__half_as_ushort(src[2 * k]) | (uint32_t)__half_as_ushort(src[2 * k + 1]) << 16;
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (p.scale_log2 < 0) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
            }
            *reinterpret_cast<uint4*>(place(r, col)) = v;
            if constexpr (SPLIT) *reinterpret_cast<uint4*>(place(r, col) + QB) = make_uint4(0, 0, 0, 0);
            if (SPLIT && col == 0) sh.down[r] = 1.f;
        }
    }
    proxy_fence_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase) {
        if (ok && !mbar_wait(bar, phase & 1)) {
            ok = false;
            report_error(ZTQ_ERR_TMEM_WAIT);
        }
        return ok;
    };

    if (warp >= 8 && warp < kTcaMma) {
        // ------------------------------------------------ codes -> operands: one half of the warps K, the other V
        const bool is_k = warp < 8 + kTcaConv;
        const int w = (warp - 8) % kTcaConv * kTcaGroups;         // first of the warp's groups of 16 keys
        const int* table = p.block_table + (long long)it.b * p.width;
        constexpr int KL = D / 64, LR = D / 4, VG = LR / 16;      // 16-byte loads per key and lane; lanes per row of V, key groups per lane
        const int vg = lane / LR, vd = lane % LR;                 // V: first key group, word of four dims
        const int rot = (vd >> 1) & 3;
        auto sel = [](int a, int b) { return (uint32_t)(a | (4 + a) << 4 | b << 8 | (4 + b) << 12); };
        const uint32_t sel0 = sel(rot, (rot + 1) & 3), sel1 = sel((rot + 2) & 3, (rot + 3) & 3);
        uint64_t* full = is_k ? sh.k_full : sh.v_full;
        uint64_t* empty = is_k ? sh.k_empty : sh.v_empty;
        const float* scales = is_k ? p.ks : p.vs;
        const int8_t* codes = is_k ? p.kc : p.vc;
        // every lane looks up group (lane & 7): all groups' blocks and scales are known to all warps
        auto look = [&](int kt) {
            const int tok = kt * kTcaKeys + 16 * (lane & 7);
            int blk = -1;
            if (kt < kt1 && attn_in_span(tok, it.lo, it.hi, p.shift)) {
                blk = table[tok >> p.shift];
                if ((unsigned)blk >= (unsigned)p.blocks) {
                    report_error(ZTQ_ERR_BLOCK);
                    blk = -1;
                }
            }
            return blk;
        };
        auto scale_of = [&](int blk) { return blk >= 0 ? scales[(long long)blk * p.kv_heads + it.h] : 0.f; };
        uint4 raw[kTcaGroups][2 * KL];                            // 16 keys' codes of this lane, for every group
        auto load = [&](int kt, int blks) {
#pragma unroll
            for (int g = 0; g < kTcaGroups; ++g) {
                const int own = __shfl_sync(0xffffffffu, blks, w + g);
                const int at = (kt * kTcaKeys + 16 * (w + g)) & ((1 << p.shift) - 1);
                const int8_t* src = codes + max(own, 0) * p.block_stride + (((long long)it.h << p.shift) + at) * D;
                if (own < 0) {
#pragma unroll
                    for (int i = 0; i < 2 * KL; ++i) raw[g][i] = make_uint4(0, 0, 0, 0);
                } else if (is_k) {                                // key (lane & 7) + 8 a, piece lane / 8 + 4 j
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int j = 0; j < KL; ++j) raw[g][a * KL + j] = ld_stream(src + ((lane & 7) + 8 * a) * D + 16 * ((lane >> 3) + 4 * j));
                } else {                                          // four dims of eight keys, VG times
                    uint32_t* r = reinterpret_cast<uint32_t*>(&raw[g][0]);
#pragma unroll
                    for (int v = 0; v < VG; ++v)
#pragma unroll
                        for (int i = 0; i < 8; ++i) r[8 * v + i] = __ldg(reinterpret_cast<const uint32_t*>(src + (8 * (vg + v) + i) * D + 4 * vd));
                }
            }
        };
        int blk = look(kt0), blk1 = look(kt0 + 1);
        float sc = scale_of(blk);
        if (n > 0) load(kt0, blk);
        for (int i = 0; i < n; ++i) {
            const int slot = i & 1;
            const int blk2 = look(kt0 + i + 2);                   // two steps ahead, scales one: their loads wait for one another
            const float sc1 = scale_of(blk1);
            // factors of the step
            const bool fine = fabsf(sc) <= 3.402823466e38f;
            TcaInfo& f = sh.info[i & 3];
            if (warp == 8) {
                if (lane < 8) f.ks[lane] = fabsf(attn_k_scale(sc));
                const uint32_t hidden = __ballot_sync(0xffffffffu, blk < 0) & 255u;
                if (lane == 0) f.hidden = hidden;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.info_full[i & 3]);
            } else if (warp == 8 + kTcaConv) {
                const uint32_t bad = __ballot_sync(0xffffffffu, blk >= 0 && !fine) & 255u;
                if (lane < 8) { f.vs[lane] = fine ? sc : 0.f; f.ve[lane] = fine ? attn_exponent(sc) : (float)kAttnLeast; }
                if (lane == 0) f.bad_v = bad;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.info_full[i & 3]);
            }
            if (i >= 2 && !wait(&empty[slot], (i >> 1) - 1)) break;
#pragma unroll
            for (int g = 0; g < kTcaGroups; ++g) {
                const bool plus = !(__shfl_sync(0xffffffffu, sc, w + g) < 0.f);      // a negative K scale turns its codes, so that the factor is positive
                if (is_k) {
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int j = 0; j < KL; ++j) {
                            const uint4 q = raw[g][a * KL + j];
                            const uint32_t x[4] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u, q.z ^ 0x80808080u, q.w ^ 0x80808080u};
                            uint32_t o[8];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                o[2 * k] = turned(__byte_perm(x[k], 0x64646464u, 0x4140), plus);
                                o[2 * k + 1] = turned(__byte_perm(x[k], 0x64646464u, 0x4342), plus);
                            }
                            uint8_t* d = sk + slot * KB + (2 * (w + g) + a) * (CG * 128) + 2 * ((lane >> 3) + 4 * j) * 128 + (lane & 7) * 16;
                            *reinterpret_cast<uint4*>(d) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(d + 128) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                } else {
                    // transposed: eight keys of one dim are 16 bytes; the lane's four dims in an order that spreads the banks
                    const uint32_t* q = reinterpret_cast<const uint32_t*>(&raw[g][0]);
#pragma unroll
                    for (int v = 0; v < VG; ++v) {
                        uint32_t o[4][4];                         // [dim slot][pair of keys]
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t x = q[8 * v + 2 * k] ^ 0x80808080u, y = q[8 * v + 2 * k + 1] ^ 0x80808080u;
                            const uint32_t u0 = __byte_perm(x, y, sel0), u1 = __byte_perm(x, y, sel1);
                            o[0][k] = unbias(__byte_perm(u0, 0x64646464u, 0x4140));
                            o[1][k] = unbias(__byte_perm(u0, 0x64646464u, 0x4342));
                            o[2][k] = unbias(__byte_perm(u1, 0x64646464u, 0x4140));
                            o[3][k] = unbias(__byte_perm(u1, 0x64646464u, 0x4342));
                        }
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const int dim = 4 * vd + ((d + rot) & 3);
                            *reinterpret_cast<uint4*>(sv + slot * KB + (dim >> 3) * (kTcaKeys / 8 * 128) + (2 * (w + g) + vg + v) * 128 + (dim & 7) * 16) = make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
                        }
                    }
                }
            }
            proxy_fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
            if (i + 1 < n) load(kt0 + i + 1, blk1);
            blk = blk1; blk1 = blk2; sc = sc1;
        }
    } else if (warp == kTcaMma) {
        // ------------------------------------------------ products
        if (elect_one()) {
            const uint32_t id_s = tc_idesc_f16(kTcaKeys), id_o = tc_idesc_f16(D);
            auto scores = [&](int t, int i) {
                const uint64_t a = tc_smem_desc(sq + t * QB, 128, CG * 128), b = tc_smem_desc(sk + (i & 1) * KB, 128, CG * 128);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) tc_mma_f16(tmem + kS + 128 * t, a + 16 * k, b + 16 * k, id_s, k > 0);
                if constexpr (SPLIT) {
                    const uint64_t rest = tc_smem_desc(sq + QB, 128, CG * 128);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) tc_mma_f16(tmem + kS, rest + 16 * k, b + 16 * k, id_s, 1);
                }
                tc_commit(&sh.s_full[t]);
            };
            if (n > 0 && wait(&sh.k_full[0], 0)) {
                tc_fence_after();
                for (int t = 0; t < tiles; ++t) scores(t, 0);
                tc_commit(&sh.k_empty[0]);
            }
            for (int i = 0; i < n && ok; ++i) {
                if (!wait(&sh.v_full[i & 1], i >> 1)) break;
                if (i + 1 < n && !wait(&sh.k_full[(i + 1) & 1], (i + 1) >> 1)) break;
                for (int t = 0; t < tiles; ++t) {
                    if (!wait(&sh.p_full[t], i)) break;
                    tc_fence_after();
                    const uint64_t b = tc_smem_desc(sv + (i & 1) * KB, 128, kTcaKeys / 8 * 128);
#pragma unroll
                    for (int k = 0; k < kTcaKeys / 16; ++k) tc_mma_f16_ta(tmem + kO + D * t, tmem + kS + 128 * t + 8 * k, b + 16 * k, id_o, i > 0 || k > 0);
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int k = 0; k < kTcaKeys / 16; ++k) tc_mma_f16_ta(tmem + kO, tmem + kS + 128 + 8 * k, b + 16 * k, id_o, 1);
                    }
                    if (t == tiles - 1) tc_commit(&sh.v_empty[i & 1]);
                    if (i + 1 < n) {
                        scores(t, i + 1);
                        if (t == tiles - 1) tc_commit(&sh.k_empty[(i + 1) & 1]);
                    } else tc_commit(&sh.o_full[t]);
                }
            }
        }
        __syncwarp();
    } else if (warp < 8 && (warp >> 2) < tiles) {
        // ------------------------------------------------ softmax: a thread is a row
        const int t = warp >> 2, r = it.r0 + 128 * t + (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);         // TMEM address: lane << 16 | column
        const uint32_t s_at = lanes + kS + 128 * t, o_at = lanes + kO + D * t;
        const bool live = r < it.r1;
        const int base = it.s.len - it.s.fresh;
        const int z = live ? min(base + r / p.group, it.s.len - 1) : -1;    // last key the row sees
        const int z_lo = p.window > 0 ? z - p.window : -1;                  // the last one in front of those it sees
        const float scale = fabsf(p.scale_log2), down = SPLIT ? sh.down[r - it.r0] : 1.f;
        float m = -INFINITY, l = 0.f, shift = 0.f;              // the reference c, the sum of the weights, what exponents are moved by
        for (int i = 0; i < n; ++i) {
            if (!wait(&sh.info_full[i & 3], i >> 2) || !wait(&sh.s_full[t], i)) break;
            tc_fence_after();
            const TcaInfo& info = sh.info[i & 3];
            const int key0 = (kt0 + i) * kTcaKeys;
            // keys of the step that the row sees: columns (a, b], less hidden groups
            const int a = z_lo - key0, b = z - key0;
            const bool edge = __any_sync(0xffffffffu, a >= 0 || b < kTcaKeys - 1) || info.hidden;
            auto seen = [&](int col) { return col <= b && col > a && !(info.hidden >> (col >> 4) & 1); };
            // f(chunk, its sixteen scores: those of a group of keys), the next chunk on its way meanwhile
            auto scores = [&](auto f) {
                uint32_t r[2][16];
                tc_ld16_nowait(s_at, r[0]);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    tc_wait16(r[c & 1]);
                    if (c < 7) tc_ld16_nowait(s_at + 16 * (c + 1), r[(c + 1) & 1]);
                    f(c, r[c & 1]);
                }
            };
            float tops[8];                                      // of the groups
            auto highest = [&](auto masked) {
                scores([&](int c, const uint32_t (&r)[16]) {
                    float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};         // four chains
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        float x = __uint_as_float(r[k]), y = __uint_as_float(r[k + 1]);
                        if constexpr (decltype(masked)::value) {
                            x = seen(16 * c + k) ? x : -INFINITY;
                            y = seen(16 * c + k + 1) ? y : -INFINITY;
                        }
                        t4[k >> 1 & 3] = fmaxf(t4[k >> 1 & 3], fmaxf(x, y));
                    }
                    tops[c] = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                });
            };
            if (edge) highest(std::true_type());
            else highest(std::false_type());
            float fk[8], top = -INFINITY;                       // the factors are read once: between the TMEM loads they would be waited for
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                fk[c] = info.ks[c] * scale;
                if constexpr (SPLIT) fk[c] *= down;
                top = tops[c] != -INFINITY ? fmaxf(top, tops[c] * fk[c] + info.ve[c]) : top;        // -inf may meet a factor of 0
            }
            if (__any_sync(0xffffffffu, top > m + attn_slack(SPLIT))) {
                const float m_new = fmaxf(m, top);
                const AttnStep by(m, m_new);
                const float fix = by.products();
                l = by.sum(l);
                shift = attn_shift(SPLIT, m_new);
                if (i > 0) {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float o[32];
                        tc_ld32(o_at + 32 * c, o);
                        uint32_t u[16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(o[16 * h + k] * fix);
                            tc_st16(o_at + 32 * c + 16 * h, u);
                        }
                    }
                }
                m = m_new;
            }
            f2 sums[2] = {{0.f, 0.f}, {0.f, 0.f}};
            float fv[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) fv[c] = info.vs[c];
            auto weights = [&](auto masked) {
                scores([&](int c, const uint32_t (&r)[16]) {
                    const float f = fk[c], v = fv[c];
                    uint32_t u[8];
                    [[maybe_unused]] uint32_t rest[SPLIT ? 8 : 1];
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const f2 x = ffma2(f2{__uint_as_float(r[k]), __uint_as_float(r[k + 1])}, f2{f, f}, f2{shift, shift});
                        float e0 = ex2(x.x), e1 = ex2(x.y);
                        if constexpr (decltype(masked)::value) {
                            e0 = seen(16 * c + k) ? e0 : 0.f;
                            e1 = seen(16 * c + k + 1) ? e1 : 0.f;
                        }
                        sums[k >> 1 & 1] = fadd2(sums[k >> 1 & 1], f2{e0, e1});
                        const f2 w = ffma2(f2{e0, e1}, f2{v, v}, f2{0.f, 0.f});
                        u[k >> 1] = pack_half2(w.x, w.y);
                        if constexpr (SPLIT) rest[k >> 1] = pack_rest(w.x, w.y, u[k >> 1]);
                    }
                    tc_st8(s_at + 8 * c, u);                    // over scores that were read
                    if constexpr (SPLIT) tc_st8(s_at + 128 + 8 * c, rest);
                });
            };
            if (edge) weights(std::true_type());
            else weights(std::false_type());
            l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
            if (info.bad_v)
                for (int g = 0; g < 8; ++g)                     // a V scale that is not finite: NaN for the rows that see its keys
                    if (info.bad_v >> g & 1 && max(16 * g, a + 1) <= min(16 * g + 15, b)) l = __int_as_float(0x7fc00000);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.p_full[t]);
        }
        if (n > 0 && wait(&sh.o_full[t], 0)) tc_fence_after();
        // ---- the row's output, or its part
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        float* part = tp.parts + (((long long)blockIdx.x * tp.splits + blockIdx.y) * tca_rows(SPLIT) + (r - it.r0)) * (D + 2);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            float o[32];
            if (n > 0 && ok) tc_ld32(o_at + 32 * c, o);
            else {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = 0.f;
            }
            if (!live || !ok) continue;
            if (tp.splits > 1) {
#pragma unroll
                for (int k = 0; k < 32; k += 2) *reinterpret_cast<float2*>(part + 32 * c + k) = make_float2(o[k], o[k + 1]);
            } else {
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = o[k + e] * inv;
                    attn_store8(p, it.s, r, it.h, 32 * c + k, v);
                }
            }
        }
        if (live && ok && tp.splits > 1) { part[D] = m; part[D + 1] = l; }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kTcaMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Adds the ranges of an item in order: a warp per row, blockIdx.x the item, blockIdx.y eight of its rows.
template <int D>
__global__ void __launch_bounds__(256) attn_tc_join_kernel(const TcaParams tp) {
    extern __shared__ int tca_upto[];
    __shared__ int part[8];
    const AttnParams& p = tp.a;
    grid_dep_launch();
    grid_dep_wait();
    tca_scan(p, tp.rows, tca_upto, part);
    TcaItem it;
    if (!tca_item(p, tp.rows, tca_upto, blockIdx.x, it)) return;
    const int lane = threadIdx.x & 31, r = it.r0 + blockIdx.y * 8 + (threadIdx.x >> 5);
    if (r >= it.r1) return;
    float top = -INFINITY;
    auto row_of = [&](int u) { return tp.parts + (((long long)blockIdx.x * tp.splits + u) * tp.rows + (r - it.r0)) * (D + 2); };
    for (int u = 0; u < tp.splits; ++u) top = fmaxf(top, row_of(u)[D]);
    float sum = 0.f, v[D / 32] = {};
    for (int u = 0; u < tp.splits; ++u) {
        const float* row = row_of(u);
        const AttnStep by(row[D], top);
        const float fix = by.products();
        sum += by.sum(row[D + 1]);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) v[k] += fix * row[32 * k + lane];
    }
#pragma unroll
    for (int k = 0; k < D / 32; ++k) attn_store(p, it.s, r, it.h, 32 * k + lane, sum > 0.f || sum != sum ? v[k] / sum : 0.f);
}

}  // namespace ztq
