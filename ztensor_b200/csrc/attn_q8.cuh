// attn_q8.cuh -- attention of a step's queries over the paged 8-bit cache.
//
//   y_i = sum_j p_ij sv_j cv_j,   p_ij = softmax_j(scale q_i . sk_j ck_j)   over the keys j a query may see:
//   j <= position of i, j > position of i - window (window > 0).  A query that sees nothing gets zeros.
// ck, cv: int8 codes [block][kv head][token][dim]; sk, sv: one scale per (block, kv head).
//
// attn_rows_kernel: a row is a (token, query head) pair; the rows of a sequence that share a kv head are multiplied
// together, 8 NT of them at a time, so that a block of the cache is read once for all of them.  Bound by HBM while the
// rows of an item fit one tile (decoding, drafts).
//   S^T = K Q^T and Y^T = V^T P^T by mma.sync m16n8k16 with the TOKENS (then the dims) as M and the rows as N = 8: a
// decode step has 4 to 8 rows per kv head, which as M would waste half of every instruction and more.
//   No shared memory on the way: the contraction index may be permuted as long as both operands agree, so every lane
// loads 16 contiguous bytes of the cache at a time and has exactly the codes its fragments need.  K: lane (g, c) holds
// tokens g and g + 8 and bytes 64 l + 16 c of each.  V: lane (g, c) holds tokens 2c, 2c + 1, 2c + 8, 2c + 9 and dims
// g D/8 .. (g + 1) D/8, and pairs two tokens' codes by byte permutes.  P^T is the transposed accumulator of S^T
// (movmatrix).  A code becomes fp16 exactly: 0x6400 | (code + 128) is 1152 + code.
//   Online softmax per warp: the running maximum m moves only when some score exceeds it by more than kSlack in the
// exponent (one vote per 16 tokens instead of a reduction); p = 2^(s - m + kLift) then stays below 2^15, inside fp16,
// and a weight of 2^-21 of the largest is still a normal number.  Scores,
// maxima, sums and accumulators are fp32; p is rounded to fp16 for the second product (relative 2^-11, against fp16
// outputs with the same step).  With fp32 inputs or outputs (SPLIT) q and p go in as two fp16 terms each, 22 bits.
//   A tile of 16 tokens lies in one block (block sizes are multiples of 16), so its scales are two scalars: sk goes into
// the score's factor, sv multiplies the tile's own product before it is added up.
//
// Work: an item is (sequence, tile of rows, kv head); its keys are cut into steps of 64 tokens (16 per warp).  The steps
// of all items in order are dealt to the CTAs in equal contiguous ranges, whatever the lengths, so a long sequence is
// split and short ones are packed.  A CTA that holds part of an item leaves {max, sum, rows} in the workspace (at most
// two parts per CTA) and attn_join_kernel adds the parts in order.
#pragma once

#include "ztq_common.cuh"

namespace ztq {

constexpr int kAttnMaxSeqs = 4096;
constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
constexpr int kAttnStep = 16 * kAttnWarps;
constexpr int kAttnMinSteps = 2;                    // steps a CTA gets at least
constexpr float kAttnSlack = 8.f;                   // how far a score may exceed the running maximum before that moves
constexpr float kAttnLift = 7.f;                    // p = 2^(s - m + lift): below 2^15, and its fp16 steps end at 2^-31 of the largest

struct AttnParams {
    const void* q;
    void* y;
    long long q_token, q_head, y_token, y_head;
    const int* query_start;
    const int* kv_len;
    const int* block_table;
    const int8_t* kc;
    const int8_t* vc;
    const float* ks;
    const float* vs;
    long long block_stride;
    float* parts;                                   // [grid][2] slots of 8 NT (D + 2) floats
    int seqs, tokens, max_new, q_heads, kv_heads, group, width, shift, blocks, window;
    float scale_log2;                               // softmax scale times log2(e)
    int x_f32, y_f32, vec;
    int min_rows, max_rows;                         // sequences with more or fewer rows per kv head belong to another kernel
};

// One sequence as the kernels see it: lengths clamped to what the buffers hold.
struct AttnSeq {
    int first, fresh, len;                          // first row of q, new tokens, tokens in the cache
    __device__ __forceinline__ int rows(int group) const { return fresh * group; }
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& p, int b) {
    AttnSeq s;
    s.first = min(max(p.query_start[b], 0), p.tokens);
    s.fresh = min(max(p.query_start[b + 1], s.first), p.tokens) - s.first;
    const long long room = (long long)p.width << p.shift;
    s.len = (int)min((long long)max(p.kv_len[b], 0), room);
    if (s.fresh > p.max_new) {                      // announced wrongly: the caller's rows stay as they were
        report_error(ZTQ_ERR_LENGTH);
        s.fresh = 0;
    }
    const int r = s.fresh * p.group;
    if (r < p.min_rows || r > p.max_rows) s.fresh = 0;
    return s;
}
// Keys [lo, hi) that the rows [r0, r1) of a sequence see between them, and as steps.
__device__ __forceinline__ void attn_span(const AttnParams& p, const AttnSeq& s, int r0, int r1, int& lo, int& hi) {
    const int base = s.len - s.fresh;               // position of the first new token
    const int a = base + r0 / p.group, z = base + (r1 - 1) / p.group;
    hi = min(max(z + 1, 0), s.len);
    lo = p.window > 0 ? min(max(a - p.window + 1, 0), hi) : 0;
}
__device__ __forceinline__ int attn_steps(int lo, int hi, int step) {
    return max(1, (hi + step - 1) / step - lo / step);          // an item without keys still writes its zeros
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// the part of a pair that fp16 dropped
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack_half2(a - f.x, b - f.y);
}
// Two biased codes (code + 128) in the low bytes of the halves of `x | 0x64006400` -> two fp16 codes.
__device__ __forceinline__ uint32_t unbias(uint32_t x) {
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_stream8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// Where CTA i's range of `total` steps begins when `ctas` of them share it.
__device__ __forceinline__ long long attn_cut(long long total, int i, int ctas) { return total * i / ctas; }
__device__ __forceinline__ int attn_ctas(long long total, int grid) {
    const long long n = (total + kAttnMinSteps - 1) / kAttnMinSteps;
    return (int)max(1ll, min(n, (long long)grid));
}

// Steps of all items of a sequence for ONE kv head, rows in tiles of `tile`.
__device__ __forceinline__ long long attn_seq_steps(const AttnParams& p, const AttnSeq& s, int tile, int step) {
    long long sum = 0;
    const int rows = s.rows(p.group);
    for (int r = 0; r < rows; r += tile) {
        int lo, hi;
        attn_span(p, s, r, min(r + tile, rows), lo, hi);
        sum += attn_steps(lo, hi, step);
    }
    return sum;
}

// upto[b] = steps of sequences 0 .. b, over all kv heads.
__device__ __forceinline__ void attn_scan(const AttnParams& p, int tile, long long* upto, long long* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    long long before = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        long long v = b < p.seqs ? attn_seq_steps(p, attn_seq(p, b), tile, kAttnStep) * p.kv_heads : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        __syncthreads();
        if (lane == 31) part[warp] = v;
        __syncthreads();
        long long all = before;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) v += part[w];
            all += part[w];
        }
        if (b < p.seqs) upto[b] = before + v;
        before = all;
    }
    __syncthreads();
}

struct AttnItem {
    int b, r0, r1, h, lo, hi, steps;
    long long begin;                                // first step of the item in the order of all steps
};
// The item that holds step w.
__device__ __forceinline__ AttnItem attn_find(const AttnParams& p, int tile, const long long* upto, long long w, AttnSeq& s) {
    AttnItem it;
    int lo = 0, hi = p.seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] > w) hi = mid; else lo = mid + 1;
    }
    it.b = lo;
    it.begin = lo ? upto[lo - 1] : 0;
    s = attn_seq(p, lo);
    const int rows = s.rows(p.group);
    for (it.r0 = 0;; it.r0 += tile) {
        it.r1 = min(it.r0 + tile, rows);
        attn_span(p, s, it.r0, it.r1, it.lo, it.hi);
        it.steps = attn_steps(it.lo, it.hi, kAttnStep);
        const long long n = (long long)it.steps * p.kv_heads;
        if (w < it.begin + n || it.r1 >= rows) break;
        it.begin += n;
    }
    it.h = (int)((w - it.begin) / it.steps);
    it.begin += (long long)it.h * it.steps;
    return it;
}

__device__ __forceinline__ void attn_store(const AttnParams& p, const AttnSeq& s, int r, int h, int d, float v) {
    const long long at = (s.first + r / p.group) * p.y_token + (long long)(h * p.group + r % p.group) * p.y_head + d;
    if (p.y_f32) static_cast<float*>(p.y)[at] = v;
    else static_cast<__half*>(p.y)[at] = __float2half_rn(v);
}

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kAttnThreads, NT == 1 && D <= 128 && !SPLIT ? 4 : NT <= 2 && D <= 128 ? 2 : 1)
    attn_rows_kernel(const AttnParams p) {
    constexpr int TILE = 8 * NT, KS = D / 16, KL = D / 64;      // rows of an item, k-steps, 16-byte loads per row of K
    constexpr int VB = D / 8;                                   // dims of V per lane
    extern __shared__ __align__(16) uint8_t smem[];
    float* red = reinterpret_cast<float*>(smem);                // [warps][TILE][D + 4]: acc, then max and sum
    long long* upto = reinterpret_cast<long long*>(smem + kAttnWarps * TILE * (D + 4) * 4);
    __shared__ long long part[kAttnWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;

    grid_dep_launch();
    grid_dep_wait();
    attn_scan(p, TILE, upto, part);
    const long long total = upto[p.seqs - 1];
    const int ctas = attn_ctas(total, gridDim.x);
    if ((int)blockIdx.x >= ctas) return;
    const long long w_end = attn_cut(total, blockIdx.x + 1, ctas);

    for (long long w = attn_cut(total, blockIdx.x, ctas); w < w_end;) {
        AttnSeq s;
        const AttnItem it = attn_find(p, TILE, upto, w, s);
        const int step0 = (int)(w - it.begin), step1 = (int)min((long long)it.steps, step0 + (w_end - w));
        const int rows = it.r1 - it.r0, base = s.len - s.fresh;
        const int head = it.h * p.group;

        // the item's queries as B fragments; columns are the rows r0 + 8 t + g
        uint32_t qh[NT][KS][2], ql[SPLIT ? NT : 1][KS][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = it.r0 + 8 * t + g;
            const bool live = r < it.r1;
            const long long at = live ? (s.first + r / p.group) * p.q_token + (long long)(head + r % p.group) * p.q_head : 0;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const long long d0 = at + 64 * (j / 4) + 16 * c + 4 * (j % 4);
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (live) {
                    if (p.x_f32) {
                        const float* f = static_cast<const float*>(p.q) + d0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = f[i];
                    } else if (p.vec) {
                        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __half*>(p.q) + d0);
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
                        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
                    } else {
                        const __half* f = static_cast<const __half*>(p.q) + d0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = __half2float(f[i]);
                    }
                }
                qh[t][j][0] = pack_half2(v[0], v[1]);
                qh[t][j][1] = pack_half2(v[2], v[3]);
                if constexpr (SPLIT) {
                    ql[t][j][0] = pack_rest(v[0], v[1], qh[t][j][0]);
                    ql[t][j][1] = pack_rest(v[2], v[3], qh[t][j][1]);
                }
            }
        }

        float acc[NT][KS][4];                                   // [dims 2 mt (+1) of the lane's][rows 2c, 2c + 1]
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
#pragma unroll
            for (int j = 0; j < KS; ++j) acc[t][j][0] = acc[t][j][1] = acc[t][j][2] = acc[t][j][3] = 0.f;
        }
        // last key that each of the lane's rows sees (its first is that less the window)
        int last[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = it.r0 + 8 * t + 2 * c + i;
                last[t][i] = r < it.r1 ? min(base + r / p.group, s.len - 1) : -1;
            }

        const int tok0 = (it.lo / kAttnStep + step0) * kAttnStep + 16 * warp, tok1 = min(it.hi, (it.lo / kAttnStep + step1) * kAttnStep);
        const int* table = p.block_table + (long long)it.b * p.width;
        auto block_of = [&](int tok) {
            int blk = table[tok >> p.shift];
            if ((unsigned)blk >= (unsigned)p.blocks) {
                report_error(ZTQ_ERR_BLOCK);
                blk = -1;
            }
            return blk;
        };
        const int mask = (1 << p.shift) - 1;
        uint4 kbuf[2][KL];
        uint32_t vbuf[4][VB / 4];
        int blk = tok0 < tok1 ? block_of(tok0) : -1;
        auto load_k = [&](int blk, int tok) {
            const int8_t* src = p.kc + max(blk, 0) * p.block_stride + (((long long)it.h << p.shift) + (tok & mask) + g) * D + 16 * c;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < KL; ++j) kbuf[i][j] = ld_stream(src + 8 * i * D + 64 * j);
        };
        auto load_v = [&](int blk, int tok) {
            const int8_t* src = p.vc + max(blk, 0) * p.block_stride + (((long long)it.h << p.shift) + (tok & mask) + 2 * c) * D + VB * g;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int8_t* row = src + ((i & 1) + 8 * (i >> 1)) * D;
                if constexpr (VB == 8) {
                    const uint2 u = ld_stream8(row);
                    vbuf[i][0] = u.x; vbuf[i][1] = u.y;
                } else {
#pragma unroll
                    for (int j = 0; j < VB / 16; ++j) {
                        const uint4 u = ld_stream(row + 16 * j);
                        vbuf[i][4 * j] = u.x; vbuf[i][4 * j + 1] = u.y; vbuf[i][4 * j + 2] = u.z; vbuf[i][4 * j + 3] = u.w;
                    }
                }
            }
        };
        if (tok0 < tok1) {
            load_k(blk, tok0);
            load_v(blk, tok0);
        }
        for (int tok = tok0; tok < tok1; tok += kAttnStep) {
            const int next = tok + kAttnStep;
            const int blk_next = next < tok1 ? block_of(next) : -1;
            const float ks = blk >= 0 ? p.ks[(long long)blk * p.kv_heads + it.h] : 0.f;
            float vs = blk >= 0 ? p.vs[(long long)blk * p.kv_heads + it.h] : 0.f;
            // ---- scores of 16 tokens
            float sc[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const uint4 w0 = kbuf[0][j / 4], w1 = kbuf[1][j / 4];
                const uint32_t x = (j % 4 == 0 ? w0.x : j % 4 == 1 ? w0.y : j % 4 == 2 ? w0.z : w0.w) ^ 0x80808080u;
                const uint32_t y = (j % 4 == 0 ? w1.x : j % 4 == 1 ? w1.y : j % 4 == 2 ? w1.z : w1.w) ^ 0x80808080u;
                const uint32_t a[4] = {unbias(__byte_perm(x, 0x64646464u, 0x4140)), unbias(__byte_perm(y, 0x64646464u, 0x4140)),
                                       unbias(__byte_perm(x, 0x64646464u, 0x4342)), unbias(__byte_perm(y, 0x64646464u, 0x4342))};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mma_f16(sc[t], a, qh[t][j][0], qh[t][j][1]);
                    if constexpr (SPLIT) mma_f16(sc[t], a, ql[t][j][0], ql[t][j][1]);
                }
            }
            if (next < tok1) load_k(blk_next, next);
            // ---- masks and the running maximum
            const float f = ks * p.scale_log2;
            bool grows = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = tok + g + 8 * (i >> 1), z = last[t][i & 1];
                    const bool seen = blk >= 0 && key <= z && (p.window <= 0 || key > z - p.window);
                    sc[t][i] = seen ? sc[t][i] * f : -INFINITY;
                    grows |= sc[t][i] > m[t][i & 1] + kAttnSlack;
                }
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(sc[t][i], sc[t][i + 2]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        if (top > m[t][i]) {
                            const float fix = m[t][i] == -INFINITY ? 0.f : exp2f(m[t][i] - top);
                            l[t][i] *= fix;
#pragma unroll
                            for (int j = 0; j < KS; ++j) { acc[t][j][i] *= fix; acc[t][j][i + 2] *= fix; }
                            m[t][i] = top;
                        }
                    }
            }
            // ---- p as B fragments
            uint32_t ph[NT][2], pl[SPLIT ? NT : 1][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = sc[t][i] == -INFINITY ? 0.f : exp2f(sc[t][i] - m[t][i & 1] + kAttnLift);
                    l[t][i & 1] += e[i];
                }
                const uint32_t h0 = pack_half2(e[0], e[1]), h1 = pack_half2(e[2], e[3]);
                ph[t][0] = transpose8x8(h0);
                ph[t][1] = transpose8x8(h1);
                if constexpr (SPLIT) {
                    pl[t][0] = transpose8x8(pack_rest(e[0], e[1], h0));
                    pl[t][1] = transpose8x8(pack_rest(e[2], e[3], h1));
                }
            }
            // ---- their values: four dims of four tokens at a time
            if (!(fabsf(vs) <= 3.402823466e38f)) {              // reaches the rows that see the tile, not the masked ones
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const bool sees = sc[t][i] != -INFINITY || sc[t][i + 2] != -INFINITY;
                        unsigned who = __ballot_sync(0xffffffffu, sees);
                        who |= who >> 16; who |= who >> 8; who |= who >> 4;
                        if (who >> c & 1) l[t][i] = __int_as_float(0x7fc00000);
                    }
                vs = 0.f;
            }
#pragma unroll
            for (int q4 = 0; q4 < VB / 4; ++q4) {
                const uint32_t x0 = vbuf[0][q4] ^ 0x80808080u, x1 = vbuf[1][q4] ^ 0x80808080u, x2 = vbuf[2][q4] ^ 0x80808080u, x3 = vbuf[3][q4] ^ 0x80808080u;
                const uint32_t lo01 = __byte_perm(x0, x1, 0x5140), hi01 = __byte_perm(x0, x1, 0x7362);     // dims 0, 1 | 2, 3 of both
                const uint32_t lo23 = __byte_perm(x2, x3, 0x5140), hi23 = __byte_perm(x2, x3, 0x7362);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t u = half ? hi01 : lo01, v = half ? hi23 : lo23;
                    const uint32_t a[4] = {unbias(__byte_perm(u, 0x64646464u, 0x4140)), unbias(__byte_perm(u, 0x64646464u, 0x4342)),
                                           unbias(__byte_perm(v, 0x64646464u, 0x4140)), unbias(__byte_perm(v, 0x64646464u, 0x4342))};
                    const int mt = 2 * q4 + half;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float o[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_f16(o, a, ph[t][0], ph[t][1]);
                        if constexpr (SPLIT) mma_f16(o, a, pl[t][0], pl[t][1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][mt][i] = fmaf(vs, o[i], acc[t][mt][i]);
                    }
                }
            }
            if (next < tok1) load_v(blk_next, next);
            blk = blk_next;
        }

        // ---- the warps' parts meet in shared memory
        __syncthreads();                                        // the previous segment's readers are done
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float sum = l[t][i];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                float* row = red + (warp * TILE + 8 * t + 2 * c + i) * (D + 4);
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    row[VB * g + 2 * j] = acc[t][j][i];
                    row[VB * g + 2 * j + 1] = acc[t][j][i + 2];
                }
                if (g == 0) { row[D] = m[t][i]; row[D + 1] = sum; }
            }
        __syncthreads();
        const bool whole = step0 == 0 && step1 == it.steps;
        float* out = p.parts + ((long long)blockIdx.x * 2 + (step0 == 0 ? 1 : 0)) * TILE * (D + 2);
        for (int i = tid; i < rows * D; i += kAttnThreads) {
            const int r = i / D, d = i % D;
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kAttnWarps; ++u) top = fmaxf(top, red[(u * TILE + r) * (D + 4) + D]);
            float sum = 0.f, v = 0.f;
#pragma unroll
            for (int u = 0; u < kAttnWarps; ++u) {
                const float* row = red + (u * TILE + r) * (D + 4);
                const float fix = row[D] == -INFINITY ? 0.f : exp2f(row[D] - top);
                sum += fix * row[D + 1];
                v += fix * row[d];
            }
            if (whole) attn_store(p, s, it.r0 + r, it.h, d, sum > 0.f || sum != sum ? v / sum : 0.f);
            else {
                out[r * (D + 2) + d] = v;
                if (d == 0) { out[r * (D + 2) + D] = top; out[r * (D + 2) + D + 1] = sum; }
            }
        }
        w += step1 - step0;
    }
}

// Adds the parts of the items that several CTAs shared.  blockIdx.x = j looks at the boundary between the ranges of CTAs j
// and j + 1 of attn_rows_kernel and does the item it cuts, if it is the first boundary inside that item; blockIdx.y is the
// row.  A short row of long loads: the parts' maxima and sums are fetched together, then every warp adds its share of the
// parts (all loads independent), then the warps' sums are added in order.
constexpr int kJoinThreads = 256;
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnParams p, int grid) {
    constexpr int TILE = 8 * NT, V = D / 32, WARPS = kJoinThreads / 32;   // V: dims per lane
    extern __shared__ __align__(16) uint8_t smem[];
    long long* upto = reinterpret_cast<long long*>(smem);
    float* fix = reinterpret_cast<float*>(upto + p.seqs);                  // [parts], at most one per CTA
    __shared__ long long part[WARPS];
    __shared__ float red[WARPS][D + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dep_launch();
    grid_dep_wait();
    attn_scan(p, TILE, upto, part);
    const long long total = upto[p.seqs - 1];
    const int ctas = attn_ctas(total, grid), cta = blockIdx.x, r = blockIdx.y;
    if (cta + 1 >= ctas) return;
    const long long w = attn_cut(total, cta + 1, ctas);
    AttnSeq s;
    const AttnItem it = attn_find(p, TILE, upto, w, s);
    if (it.begin == w || attn_cut(total, cta, ctas) > it.begin || r >= it.r1 - it.r0) return;     // no cut inside, or not the first one
    // CTAs cta .. cta + n - 1 hold parts; the last is the one whose range reaches the item's end
    const long long end = it.begin + it.steps;
    int last = (int)(end * ctas / total);
    while (last > cta && attn_cut(total, last, ctas) >= end) --last;
    while (attn_cut(total, last + 1, ctas) < end) ++last;
    const int n = last - cta + 1;
    auto row_of = [&](int u) { return p.parts + ((long long)(cta + u) * 2 + (u == 0 ? 1 : 0)) * TILE * (D + 2) + r * (D + 2); };
    float top = -INFINITY;
    for (int u = tid; u < n; u += kJoinThreads) {
        const float m = row_of(u)[D];
        fix[u] = m;
        top = fmaxf(top, m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[warp][0] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < WARPS; ++k) top = fmaxf(top, red[k][0]);
    __syncthreads();
    float sum = 0.f, v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
#pragma unroll 4
    for (int u = warp; u < n; u += WARPS) {
        const float* row = row_of(u);
        const float f = fix[u] == -INFINITY ? 0.f : exp2f(fix[u] - top);
        sum += f * row[D + 1];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += f * row[32 * k + lane];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) red[warp][32 * k + lane] = v[k];
    if (lane == 0) red[warp][D] = sum;
    __syncthreads();
    for (int d = tid; d < D; d += kJoinThreads) {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) { a += red[k][d]; b += red[k][D]; }
        attn_store(p, s, it.r0 + r, it.h, d, b > 0.f || b != b ? a / b : 0.f);
    }
}

}  // namespace ztq
