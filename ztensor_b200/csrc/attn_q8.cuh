// attn_q8.cuh -- attention of a step's queries over the paged 8-bit cache.
//
//   y_i = sum_j p_ij sv_j cv_j,   p_ij = softmax_j(scale q_i . sk_j ck_j)   over the keys j a query may see:
//   j <= position of i, j > position of i - window (window > 0).  A query that sees nothing gets zeros.
// ck, cv: int8 codes [block][kv head][token][dim]; sk, sv: one scale per (block, kv head).
//
// attn_rows_kernel: a row is a (token, query head) pair; the rows of a sequence that share a kv head are multiplied
// together, 8 NT of them at a time, so that a block of the cache is read once for all of them.  Bound by HBM while the
// rows of an item fit one tile (decoding, drafts).
//   One CTA per SM: a producer warp keeps a ring of steps of 128 tokens (32 KB at D = 128) filled by tiled TMA copies, one
// per block, and looks up block table and scales one step ahead; the other warps take 16 tokens of a step in turn.  Twelve of
// them where 128 registers suffice: a warp's tile is a chain of 380 instructions that eight warps leave half hidden
// (64 sequences of 3000 to 12000 tokens, 958 MB: 211 us with eight,
// 192 with twelve and the look-ahead of the producer, when it was tried).
//   S^T = K Q^T and Y^T = V^T P^T by mma.sync m16n8k16 with the TOKENS (then the dims) as M and the rows as N = 8: a
// decode step has 4 to 8 rows per kv head, which as M would waste half of every instruction and more.
//   The contraction index may be permuted as long as both operands agree, so every lane reads 16 contiguous bytes of the
// step at a time and has exactly the codes its fragments need.  K: lane (g, c) holds tokens tau(g) and tau(g) + 8 and the
// 16-byte pieces c + 4 l of each.  V: lane (g, c) holds tokens tau(2c), tau(2c + 1) and those + 8, pieces g + 8 j, and
// pairs two tokens' codes by byte permutes.  P^T is the transposed accumulator of S^T (movmatrix).  tau = 0 5 2 7 4 1 6 3:
// with the copies' 128-byte swizzle both reads are free of bank conflicts (even and odd g differ in bit 2 of the row, even
// rows of the c's are all different).  A code becomes fp16 exactly: 0x6400 | (code + 128) is 1152 + code.
//   Online softmax per warp and row, whose reference c is the largest exponent not of a weight but of a weight TIMES the power
// of two of its V scale: p = 2^(s - c + 4) sv then stays inside fp16 and ends at 2^-29 of the row's largest such product,
// whatever the scales of blocks are that the row does not see or hardly weighs.  c moves only when exceeded by more than a
// slack of 8 (one vote per 16 tokens instead of a reduction); it is not rounded, so that a weight that outweighs all others
// is exact.  The weights' sum is relative to 2^c too, which may be 2^127 apart from 1: fp32 holds that.
//   Scores, references, sums and accumulators are fp32; p is rounded to fp16 for the second product (relative 2^-11, against
// fp16 outputs with the same step).  With fp32 inputs or outputs (SPLIT) q and p go in as two fp16 terms each, 22 bits; a row
// of fp32 queries is first brought near the upper end of fp16's range by a power of two, which its scores are divided by.
//   A tile of 16 tokens lies in one block (block sizes are multiples of 16), so its scales are two scalars: sk goes into
// the score's factor, sv into p.
//
// Measured: 64 sequences of 3000 to 12000 tokens, 64 / 8 heads of 128 (958 MB) 186 to 200 us from box to box (5.15 to 4.8 TB/s),
// 160 with the arithmetic left out; one sequence of 8192 tokens 18 us with the join, of which the copies and the arithmetic take 4.
//
// Work: an item is (sequence, tile of rows, kv head).  The steps of all items in order are dealt to the CTAs in equal
// contiguous ranges, whatever the lengths, so a long sequence is split and short ones are packed.  A CTA that holds part of
// an item leaves {max, sum, rows} in the workspace (at most two parts per CTA) and attn_join_kernel adds the parts in
// order.
#pragma once

#include "tc_common.cuh"

namespace ztq {

constexpr int kAttnMaxSeqs = 4096;
constexpr int kAttnStep = 128;                      // tokens of a step: eight tiles of 16, dealt to the warps in turn
constexpr int kAttnMinSteps = 1;                    // steps a CTA gets at least
constexpr uint32_t kAttnHidden = 0xfffe5afeu;       // in place of a K scale: 16 tokens without a block (a NaN no arithmetic makes)
// The exponent of a weight's product with its V scale may exceed c by `slack`, and a scale is below twice its power of two:
// p = 2^(s - c + lift) sv < 2^(slack + lift + 1), which has to stay below 2^16.  With two terms per weight (SPLIT) more bits go to small
// weights.
__host__ __device__ constexpr float attn_slack(bool split) { return split ? 2.f : 8.f; }
__host__ __device__ constexpr float attn_lift(bool split) { return split ? 12.f : 4.f; }
static_assert(attn_slack(false) + attn_lift(false) + 1 < 16 && attn_slack(true) + attn_lift(true) + 1 < 16, "p stays in fp16");
// V scales below 2^kAttnLeast count as that: sums of weights stay below 2^(slack + lift - kAttnLeast) times their number, and products
// below 2^(kAttnLeast - 29) may vanish.
constexpr int kAttnLeast = -90;

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
    int x_f32, y_f32, vec, y_wide;                  // vec, y_wide: reads of four elements of q, 16-byte stores of y
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
    lo = p.window > 0 ? (int)min(max((long long)a - p.window + 1, 0ll), (long long)hi) : 0;
}
// Whether the block that holds token `tok` holds any of the keys [lo, hi): what lies in front of a window may have lost its block.
__device__ __forceinline__ bool attn_in_span(int tok, int lo, int hi, int shift) { return tok < hi && tok >> shift >= lo >> shift; }
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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Keys of an infinite scale are infinities of both signs and NaN: so are a row's scores.
__device__ __forceinline__ float attn_k_scale(float sk) { return fabsf(sk) <= 3.402823466e38f ? sk : __int_as_float(0x7fc00000); }
// The exponent of a finite V scale
__device__ __forceinline__ float attn_exponent(float sv) { return (float)max((int)(__float_as_uint(fabsf(sv)) >> 23) - 127, kAttnLeast); }
// What exponents are moved by for a reference
__device__ __forceinline__ float attn_shift(bool split, float c) { return c == -INFINITY ? 0.f : attn_lift(split) - c; }
// The factor 2^(from - to), from <= to, between two references in two parts: sums of weights may be more than fp32's 2^126 apart and
// matter still, products do not.  Both take the same factor, so its error of 2^-22 drops out.
struct AttnStep {
    float a, b;
    __device__ __forceinline__ AttnStep(float from, float to) {
        const float d = from - to;                          // 2^-252 also where `from`, or both, are -inf
        a = ex2(fmaxf(d, -126.f));
        b = ex2(fminf(fmaxf(d + 126.f, -126.f), 0.f));
    }
    __device__ __forceinline__ float sum(float x) const { return x * a * b; }
    __device__ __forceinline__ float products() const { return a * b; }
};
// The power of two that brings a row whose largest element is `top` to [2^14, 2^15), where two fp16 terms hold 22 bits of every element
// down to 2^-17 of the largest, and the others to 2^-39 of that (a row below 2^-112 stays below, and its subnormal numbers are exact).
__device__ __forceinline__ float attn_up(float top) { return __uint_as_float(min(127 + 14 + 127 - (__float_as_uint(top) >> 23), 253u) << 23); }
__device__ __forceinline__ float attn_down(float up) { return __uint_as_float((254u << 23) - __float_as_uint(up)); }      // its reciprocal
__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// Where CTA i's range of `total` steps begins when `ctas` of them share it.
// (divisions in 64 bits take hundreds of clocks each, and stand in front of everything else)
__device__ __forceinline__ long long attn_cut(long long total, int i, int ctas) {
    return total < (1 << 20) ? (unsigned)total * (unsigned)i / (unsigned)ctas : total * i / ctas;      // ctas < 2^12
}
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
    const long long ahead = w - it.begin;
    it.h = ahead < 0x7fffffff ? (int)((unsigned)ahead / (unsigned)it.steps) : (int)(ahead / it.steps);
    it.begin += (long long)it.h * it.steps;
    return it;
}

__device__ __forceinline__ void attn_store(const AttnParams& p, const AttnSeq& s, int r, int h, int d, float v) {
    const long long at = (s.first + r / p.group) * p.y_token + (long long)(h * p.group + r % p.group) * p.y_head + d;
    if (p.y_f32) static_cast<float*>(p.y)[at] = v;
    else static_cast<__half*>(p.y)[at] = __float2half_rn(v);
}

__device__ __forceinline__ void attn_store8(const AttnParams& p, const AttnSeq& s, int r, int h, int d, const float (&v)[8]) {
    const long long at = (s.first + r / p.group) * p.y_token + (long long)(h * p.group + r % p.group) * p.y_head + d;
    if (p.y_f32) {
        float* y = static_cast<float*>(p.y) + at;
        if (p.y_wide) {
            *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(y + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = v[k];
        }
    } else {
        __half* y = static_cast<__half*>(p.y) + at;
        if (p.y_wide) *reinterpret_cast<uint4*>(y) = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __float2half_rn(v[k]);
        }
    }
}

// Shared memory of a rows CTA: the ring, the exchange between its warps, the steps' factors and the scan.
template <int D, int NT, bool SPLIT>
struct AttnRing {
    static constexpr int kWarps = NT == 1 && D <= 128 && !SPLIT ? 12 : 8;      // and the producer
    static constexpr int kThreads = 32 * kWarps + 32;
    static constexpr int kStepBytes = 2 * kAttnStep * D;                       // K then V
    static constexpr int kStages = D == 64 ? 8 : D == 128 ? (NT == 1 ? 5 : 4) : 2;
    static constexpr int kSwapBytes = kWarps / 2 * 32 * (NT * D / 16 * 4 + 4 * NT) * 4;
    static constexpr int kInfo = kStages * kAttnStep / 16;                     // {sk, sv} of every 16 tokens
    static constexpr int kSwapAt = kStages * kStepBytes, kInfoAt = kSwapAt + kSwapBytes, kBarAt = kInfoAt + kInfo * 8, kScanAt = kBarAt + 2 * kStages * 8 + 16;
    static constexpr int bytes(int seqs) { return kScanAt + seqs * 8 + 1024; }  // 1024: the ring starts on the swizzle's period
};

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(AttnRing<D, NT, SPLIT>::kThreads, 1) attn_rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const AttnParams p) {
    using Ring = AttnRing<D, NT, SPLIT>;
    constexpr int kAttnWarps = Ring::kWarps;
    constexpr int TILE = 8 * NT, KS = D / 16, KL = D / 64;      // rows of an item, k-steps, 16-byte pieces of a row of K per lane
    constexpr int VB = D / 8;                                   // dims of V per lane
    constexpr int ROW = D < 128 ? D : 128;                      // bytes of a row in a swizzled tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    float* swap = reinterpret_cast<float*>(smem + Ring::kSwapAt);
    float2* info = reinterpret_cast<float2*>(smem + Ring::kInfoAt);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Ring::kBarAt);
    uint64_t* empty = full + Ring::kStages;
    long long* upto = reinterpret_cast<long long*>(smem + Ring::kScanAt);
    __shared__ long long part[kAttnWarps + 1];
    __shared__ int failed;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;

    if (tid == 32 * kAttnWarps) {                               // the maps are on their way while the lengths are read
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&k_map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < Ring::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kAttnWarps);
        }
        failed = 0;
        mbar_fence_init();
    }
    grid_dep_wait();
    grid_dep_launch();                                          // behind the wait: the join reads the lengths before its own
    attn_scan(p, TILE, upto, part);
    const long long total = upto[p.seqs - 1];
    const int ctas = attn_ctas(total, gridDim.x);
    if ((int)blockIdx.x >= ctas) return;
    const long long w0 = attn_cut(total, blockIdx.x, ctas), w_end = attn_cut(total, blockIdx.x + 1, ctas);

    if (warp == kAttnWarps) {
        // ------------------------------------------------ producer: lane 8 k + j looks after tokens 16 j .. of the k-th of four
        // steps; their blocks and scales are fetched while the four before are issued (two loads that wait for one another
        // would otherwise take as long as a step's copies)
        const int per = 1 << (p.shift - 4);                     // 16-token groups of a block: the first of them in a step copies
        int n = 0;                                              // steps issued
        for (long long w = w0; w < w_end;) {
            AttnSeq s;
            const AttnItem it = attn_find(p, TILE, upto, w, s);
            const int step0 = (int)(w - it.begin), step1 = (int)min((long long)it.steps, step0 + (w_end - w));
            const int* table = p.block_table + (long long)it.b * p.width;
            auto look = [&](int first) {                        // the block of this lane's group, -1 where there is none
                const int step = first + (lane >> 3), tok = (it.lo / kAttnStep + step) * kAttnStep + 16 * (lane & 7);
                int blk = -1;
                if (step < step1 && attn_in_span(tok, it.lo, it.hi, p.shift)) {
                    blk = table[tok >> p.shift];
                    if ((unsigned)blk >= (unsigned)p.blocks) {
                        report_error(ZTQ_ERR_BLOCK);
                        blk = -1;
                    }
                }
                return blk;
            };
            auto scales = [&](int blk) {
                const long long at = (long long)max(blk, 0) * p.kv_heads + it.h;
                return blk < 0 ? make_float2(__uint_as_float(kAttnHidden), 0.f) : make_float2(attn_k_scale(p.ks[at]), p.vs[at]);
            };
            int blk = look(step0);
            float2 f = scales(blk), f_next = f;
            for (int first = step0; first < step1; first += 4) {
                const int blk_next = look(first + 4);
                for (int k = 0; k < 4 && first + k < step1; ++k, ++n) {
                    if (k == 2) f_next = scales(blk_next);
                    const int stage = n % Ring::kStages;
                    if (n >= Ring::kStages && !mbar_wait(&empty[stage], ((n / Ring::kStages) - 1) & 1)) {
                        report_error(ZTQ_ERR_EMPTY_WAIT);
                        return;
                    }
                    const bool mine = (lane >> 3) == k, copies = mine && blk >= 0 && (lane & 7 & (per - 1)) == 0;
                    const unsigned who = __ballot_sync(0xffffffffu, copies);
                    if (copies) {                               // ahead of the arrival, which keeps the phase open: the factors may still be on their way
                        uint8_t* dst = smem + stage * Ring::kStepBytes + 16 * (lane & 7) * ROW;
                        const int row = it.h << p.shift;
#pragma unroll
                        for (int x = 0; x < D; x += 128) {
                            tma_load_3d(dst + x * kAttnStep, &k_map, x, row, blk, &full[stage]);
                            tma_load_3d(dst + kAttnStep * D + x * kAttnStep, &v_map, x, row, blk, &full[stage]);
                        }
                    }
                    if (mine) info[stage * 8 + (lane & 7)] = f;
                    __syncwarp();                               // the factors are written before lane 0 arrives
                    if (lane == 0) mbar_expect_tx(&full[stage], __popc(who) * 2 * ((16 * D) << (p.shift - 4)));
                }
                blk = blk_next; f = f_next;
            }
            w += step1 - step0;
        }
        return;
    }

    // ------------------------------------------------ the other warps
    // tau(g); tokens of the lane's V rows; byte offsets of its pieces inside its 16 tokens of a step
    const int tau = (g & 1) ? (g + 4) & 7 : g, tv0 = 2 * c, tv1 = (2 * c + 5) & 7;
    auto piece = [](int row, int chunk) {                       // 16-byte piece `chunk` of a row, as the copies swizzle it
        return D == 64 ? row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4) : (chunk >> 3) * (kAttnStep * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
    };
    int n = 0, mine = warp;                                     // steps so far; the warp's tile of the next one
    for (long long w = w0; w < w_end;) {
        AttnSeq s;
        const AttnItem it = attn_find(p, TILE, upto, w, s);
        const int step0 = (int)(w - it.begin), step1 = (int)min((long long)it.steps, step0 + (w_end - w));
        const int base = s.len - s.fresh, head = it.h * p.group;

        // the item's queries as B fragments; columns are the rows r0 + 8 t + g
        uint32_t qh[NT][KS][2], ql[SPLIT ? NT : 1][KS][2];
        [[maybe_unused]] float down[SPLIT ? NT : 1][2];         // fp32 queries: what the scores of rows 2c, 2c + 1 are multiplied by
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = it.r0 + 8 * t + g;
            const bool live = r < it.r1;
            const long long at = (live ? (s.first + r / p.group) * p.q_token + (long long)(head + r % p.group) * p.q_head : 0) + 16 * c;
            if constexpr (SPLIT) {
                float up = 1.f;
                if (p.x_f32) {
                    float v[KS][4], top = 0.f;
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[j][i] = live ? static_cast<const float*>(p.q)[at + 64 * (j / 4) + 4 * (j % 4) + i] : 0.f;
                            top = fmaxf(top, fabsf(v[j][i]));
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));        // the row's other pieces
                    up = attn_up(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float x = v[j][2 * i] * up, y = v[j][2 * i + 1] * up;
                            qh[t][j][i] = pack_half2(x, y);
                            ql[t][j][i] = pack_rest(x, y, qh[t][j][i]);
                        }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) down[t][i] = attn_down(__shfl_sync(0xffffffffu, up, 4 * (2 * c + i)));
                if (p.x_f32) continue;
            }
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const long long d0 = at + 64 * (j / 4) + 4 * (j % 4);
                uint2 u = make_uint2(0, 0);
                if (live) {
                    if (p.vec) {
                        u = *reinterpret_cast<const uint2*>(static_cast<const __half*>(p.q) + d0);
                    } else {
                        const unsigned short* f = static_cast<const unsigned short*>(p.q) + d0;
                        u = make_uint2(f[0] | (uint32_t)f[1] << 16, f[2] | (uint32_t)f[3] << 16);
                    }
                }
                qh[t][j][0] = u.x;
                qh[t][j][1] = u.y;
                if constexpr (SPLIT) ql[t][j][0] = ql[t][j][1] = 0u;
            }
        }

        float acc[NT][KS][4];                                   // [dims 2 mt (+1) of the lane's][rows 2c, 2c + 1]
        float m[NT][2], l[NT][2];                               // the references c and the sums of the weights
        int last[NT][2], z_min = 0x7fffffff, z_max = -1;        // last key that each of the lane's rows sees (its first is that less the window)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
#pragma unroll
            for (int j = 0; j < KS; ++j) acc[t][j][0] = acc[t][j][1] = acc[t][j][2] = acc[t][j][3] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = it.r0 + 8 * t + 2 * c + i;
                last[t][i] = r < it.r1 ? min(base + r / p.group, s.len - 1) : -1;
                if (r < it.r1) { z_min = min(z_min, last[t][i]); z_max = max(z_max, last[t][i]); }
            }
        }
        z_min = __reduce_min_sync(0xffffffffu, z_min);
        z_max = __reduce_max_sync(0xffffffffu, z_max);

        // The CTA's tiles are dealt to the warps in turn, eight per step: `mine` is this warp's tile of the step, if below 8.
        // A warp without one waits and arrives all the same: a barrier's parity says which phase it is in only to those
        // who have seen every phase before it.
        for (int step = step0; step < step1; ++step, ++n) {
            const int stage = n % Ring::kStages, sub = mine, tok = (it.lo / kAttnStep + step) * kAttnStep + 16 * sub;
            mine += mine < 8 ? kAttnWarps - 8 : -8;
            bool came = !*(volatile int*)&failed;
            if (came && !mbar_wait(&full[stage], (n / Ring::kStages) & 1)) {
                report_error(ZTQ_ERR_FULL_WAIT);
                *(volatile int*)&failed = 1;
                came = false;
            }
            came = __all_sync(0xffffffffu, came);
            if (sub >= 8 || tok >= it.hi || !came) {            // nothing for this warp
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
                continue;
            }
            const uint8_t* sk = smem + stage * Ring::kStepBytes + 16 * sub * ROW;
            const uint8_t* sv = sk + kAttnStep * D;
            const float2 f2 = info[stage * 8 + sub];
            const bool hidden = __float_as_uint(f2.x) == kAttnHidden;
            // ---- scores of 16 tokens, two chains
            float sc[NT][4], sd[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[t][i] = sd[t][i] = 0.f;
#pragma unroll
            for (int l4 = 0; l4 < KL; ++l4) {
                const uint4 a4 = *reinterpret_cast<const uint4*>(sk + piece(tau, c + 4 * l4)), b4 = *reinterpret_cast<const uint4*>(sk + piece(tau + 8, c + 4 * l4));
                const uint32_t xs[4] = {a4.x, a4.y, a4.z, a4.w}, ys[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = 4 * l4 + k;
                    const uint32_t x = xs[k] ^ 0x80808080u, y = ys[k] ^ 0x80808080u;
                    const uint32_t a[4] = {unbias(__byte_perm(x, 0x64646464u, 0x4140)), unbias(__byte_perm(y, 0x64646464u, 0x4140)),
                                           unbias(__byte_perm(x, 0x64646464u, 0x4342)), unbias(__byte_perm(y, 0x64646464u, 0x4342))};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_f16(j & 1 ? sd[t] : sc[t], a, qh[t][j][0], qh[t][j][1]);
                        if constexpr (SPLIT) mma_f16(j & 1 ? sc[t] : sd[t], a, ql[t][j][0], ql[t][j][1]);
                    }
                }
            }
            // ---- masks and the reference
            const float f = f2.x * p.scale_log2;
            const bool whole_tile = !hidden && tok + 15 <= z_min && (p.window <= 0 || tok > z_max - p.window);
            const bool fine = fabsf(f2.y) <= 3.402823466e38f;
            const float sv_exp = fine ? attn_exponent(f2.y) : (float)kAttnLeast;
            bool grows = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[t][i] = (sc[t][i] + sd[t][i]) * (SPLIT ? f * down[SPLIT ? t : 0][i & 1] : f);
                    if (!whole_tile) {
                        const int key = tok + tau + 8 * (i >> 1), z = last[t][i & 1];
                        const bool seen = !hidden && key <= z && (p.window <= 0 || key > z - p.window);
                        sc[t][i] = seen ? sc[t][i] : -INFINITY;
                    }
                    grows |= sc[t][i] > m[t][i & 1] + (attn_slack(SPLIT) - sv_exp);
                }
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(sc[t][i], sc[t][i + 2]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        top += sv_exp;
                        if (m[t][i] == -INFINITY) m[t][i] = top;        // nothing summed yet
                        else if (top > m[t][i]) {
                            const AttnStep by(m[t][i], top);
                            const float fix = by.products();
                            l[t][i] = by.sum(l[t][i]);
#pragma unroll
                            for (int j = 0; j < KS; ++j) { acc[t][j][i] *= fix; acc[t][j][i + 2] *= fix; }
                            m[t][i] = top;
                        }
                    }
            }
            const float sv_fine = fine ? f2.y : 0.f;
            if (!fine) {                                        // NaN for the rows that see the tile, not for the masked ones
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        unsigned sees = __ballot_sync(0xffffffffu, sc[t][i] != -INFINITY || sc[t][i + 2] != -INFINITY);
                        sees |= sees >> 16; sees |= sees >> 8; sees |= sees >> 4;
                        if (sees >> c & 1) l[t][i] = __int_as_float(0x7fc00000);
                    }
            }
            // ---- p as B fragments
            uint32_t ph[NT][2], pl[SPLIT ? NT : 1][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float shift0 = attn_shift(SPLIT, m[t][0]), shift1 = attn_shift(SPLIT, m[t][1]);
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = ex2(sc[t][i] + (i & 1 ? shift1 : shift0));
                    l[t][i & 1] += e[i];
                    e[i] *= sv_fine;
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
#pragma unroll
            for (int v4 = 0; v4 < (VB + 15) / 16; ++v4) {
                uint32_t vb[4][VB < 16 ? 2 : 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = (i & 1 ? tv1 : tv0) + 8 * (i >> 1);
                    if constexpr (VB < 16) {
                        const uint2 u = *reinterpret_cast<const uint2*>(sv + piece(row, g >> 1) + 8 * (g & 1));
                        vb[i][0] = u.x; vb[i][1] = u.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4*>(sv + piece(row, g + 8 * v4));
                        vb[i][0] = u.x; vb[i][1] = u.y; vb[i][2] = u.z; vb[i][3] = u.w;
                    }
                }
#pragma unroll
                for (int q4 = 0; q4 < (VB < 16 ? 2 : 4); ++q4) {
                    const uint32_t x0 = vb[0][q4] ^ 0x80808080u, x1 = vb[1][q4] ^ 0x80808080u, x2 = vb[2][q4] ^ 0x80808080u, x3 = vb[3][q4] ^ 0x80808080u;
                    const uint32_t lo01 = __byte_perm(x0, x1, 0x5140), hi01 = __byte_perm(x0, x1, 0x7362);     // dims 0, 1 | 2, 3 of both
                    const uint32_t lo23 = __byte_perm(x2, x3, 0x5140), hi23 = __byte_perm(x2, x3, 0x7362);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t u = half ? hi01 : lo01, v = half ? hi23 : lo23;
                        const uint32_t a[4] = {unbias(__byte_perm(u, 0x64646464u, 0x4140)), unbias(__byte_perm(u, 0x64646464u, 0x4342)),
                                               unbias(__byte_perm(v, 0x64646464u, 0x4140)), unbias(__byte_perm(v, 0x64646464u, 0x4342))};
                        const int mt = 8 * v4 + 2 * q4 + half;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            mma_f16(acc[t][mt], a, ph[t][0], ph[t][1]);
                            if constexpr (SPLIT) mma_f16(acc[t][mt], a, pl[t][0], pl[t][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
        }

        // ---- the warps' parts meet, the upper half's with the lower's until one is left, in a fixed order
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], o);
#pragma unroll
        for (int left = kAttnWarps; left > 1; left = (left + 1) / 2) {
            const int half = (left + 1) / 2;
            bar_sync(1, 32 * kAttnWarps);                       // what the exchange held before has been read
            float4* mine = reinterpret_cast<float4*>(swap) + (warp >= half ? warp - half : warp) * 32 * (NT * KS + NT) + lane;
            if (warp >= half && warp < left) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mine[32 * (NT * KS + t)] = make_float4(m[t][0], m[t][1], l[t][0], l[t][1]);
#pragma unroll
                    for (int j = 0; j < KS; ++j) mine[32 * (t * KS + j)] = make_float4(acc[t][j][0], acc[t][j][1], acc[t][j][2], acc[t][j][3]);
                }
            }
            bar_sync(1, 32 * kAttnWarps);
            if (warp + half < left) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float4 o = mine[32 * (NT * KS + t)];
                    float f0[2], f1[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float mo = i ? o.y : o.x, lo = i ? o.w : o.z;
                        const bool up = m[t][i] >= mo;                // whose reference stays
                        const AttnStep by(fminf(m[t][i], mo), fmaxf(m[t][i], mo));
                        f0[i] = up ? 1.f : by.products();
                        f1[i] = up ? by.products() : 1.f;
                        l[t][i] = up ? l[t][i] + by.sum(lo) : by.sum(l[t][i]) + lo;
                        m[t][i] = fmaxf(m[t][i], mo);
                    }
#pragma unroll
                    for (int j = 0; j < KS; ++j) {
                        const float4 x = mine[32 * (t * KS + j)];
                        acc[t][j][0] = f0[0] * acc[t][j][0] + f1[0] * x.x;
                        acc[t][j][1] = f0[1] * acc[t][j][1] + f1[1] * x.y;
                        acc[t][j][2] = f0[0] * acc[t][j][2] + f1[0] * x.z;
                        acc[t][j][3] = f0[1] * acc[t][j][3] + f1[1] * x.w;
                    }
                }
            }
        }
        if (warp == 0 && !*(volatile int*)&failed) {
            const bool whole = step0 == 0 && step1 == it.steps;
            float* out = p.parts + ((long long)blockIdx.x * 2 + (step0 == 0 ? 1 : 0)) * TILE * (D + 2);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 8 * t + 2 * c + i;
                    if (it.r0 + r >= it.r1) continue;
                    const float inv = whole ? (l[t][i] > 0.f || l[t][i] != l[t][i] ? 1.f / l[t][i] : 0.f) : 1.f;
#pragma unroll
                    for (int j = 0; j < KS; j += 4) {           // eight consecutive dims of the lane's
                        const int d = VB < 16 ? VB * g : 128 * (j / 8) + 16 * g + 2 * (j % 8);
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) { v[2 * k] = acc[t][j + k][i] * inv; v[2 * k + 1] = acc[t][j + k][i + 2] * inv; }
                        if (whole) attn_store8(p, s, it.r0 + r, it.h, d, v);
                        else {
#pragma unroll
                            for (int k = 0; k < 8; k += 2) *reinterpret_cast<float2*>(out + r * (D + 2) + d + k) = make_float2(v[k], v[k + 1]);
                        }
                    }
                    if (!whole && g == 0) *reinterpret_cast<float2*>(out + r * (D + 2) + D) = make_float2(m[t][i], l[t][i]);
                }
        }
        w += step1 - step0;
    }
}

// Adds the parts of the items that several CTAs shared: blockIdx.x = j looks at the boundary between the ranges of CTAs j and
// j + 1 of attn_rows_kernel and does the item it cuts, if it is the first boundary inside that item.  `share` warps take a
// row (all of a CTA's where items are few and have many parts): every warp adds its share of the parts, all loads
// independent, then the warps' sums are added in order.
constexpr int kJoinThreads = 256;
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnParams p, int grid) {
    constexpr int TILE = 8 * NT, V = D / 32, WARPS = kJoinThreads / 32;   // V: dims per lane
    extern __shared__ __align__(16) uint8_t smem_join[];
    long long* upto = reinterpret_cast<long long*>(smem_join);
    __shared__ long long part[WARPS];
    __shared__ float red[WARPS][D + 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dep_launch();
    attn_scan(p, TILE, upto, part);                        // the lengths are older than the kernel in front (see there)
    const long long total = upto[p.seqs - 1];
    const int ctas = attn_ctas(total, grid), cta = blockIdx.x, share = WARPS * gridDim.y / TILE;     // warps per row: 1 or WARPS
    const bool cuts = cta + 1 < ctas;
    const long long w = cuts ? attn_cut(total, cta + 1, ctas) : 0;
    AttnSeq s = {};
    AttnItem it = {};
    if (cuts) it = attn_find(p, TILE, upto, w, s);
    // Every CTA waits, also one with nothing to do: the kernel behind this one takes its end for the end of the one in front.
    grid_dep_wait();
    if (!cuts || it.begin == w || attn_cut(total, cta, ctas) > it.begin) return;     // no cut inside, or not the first one
    // CTAs cta .. cta + n - 1 hold parts; the last is the one whose range reaches the item's end
    const long long end = it.begin + it.steps;
    int last = end < (1 << 20) ? (int)((unsigned)end * (unsigned)ctas / (unsigned)total) : (int)(end * ctas / total);
    while (last > cta && attn_cut(total, last, ctas) >= end) --last;
    while (attn_cut(total, last + 1, ctas) < end) ++last;
    const int n = last - cta + 1, r = share == 1 ? blockIdx.y * WARPS + warp : blockIdx.y;
    float top = -INFINITY, sum = 0.f, v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
    if (r < it.r1 - it.r0) {
#pragma unroll 4
        for (int u = share == 1 ? 0 : warp; u < n; u += share) {
            const float* row = p.parts + ((long long)(cta + u) * 2 + (u == 0 ? 1 : 0)) * TILE * (D + 2) + r * (D + 2);
            const float2 ml = *reinterpret_cast<const float2*>(row + D);
            float x[V];
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = row[32 * k + lane];
            const bool up = top >= ml.x;                        // whose reference stays
            const AttnStep by(fminf(top, ml.x), fmaxf(top, ml.x));
            const float old = up ? 1.f : by.products(), fix = up ? by.products() : 1.f;
            sum = up ? sum + by.sum(ml.y) : by.sum(sum) + ml.y;
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = old * v[k] + fix * x[k];
            top = fmaxf(top, ml.x);
        }
    }
    if (share > 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) red[warp][32 * k + lane] = v[k];
        if (lane == 0) { red[warp][D] = top; red[warp][D + 1] = sum; }
        __syncthreads();
        if (warp) return;
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.f;
#pragma unroll
        for (int u = 0; u < WARPS; ++u) top = fmaxf(top, red[u][D]);
#pragma unroll
        for (int u = 0; u < WARPS; ++u) {
            const AttnStep by(red[u][D], top);
            const float fix = by.products();
            sum += by.sum(red[u][D + 1]);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] += fix * red[u][32 * k + lane];
        }
    }
    if (r >= it.r1 - it.r0) return;
#pragma unroll
    for (int k = 0; k < V; ++k) attn_store(p, s, it.r0 + r, it.h, 32 * k + lane, sum > 0.f || sum != sum ? v[k] / sum : 0.f);
}

}  // namespace ztq
