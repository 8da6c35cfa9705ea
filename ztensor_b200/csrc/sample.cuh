// sample.cuh -- one token per row of logits, from a given random number.
//
// With l_max the largest logit, T the temperature and the tokens ordered by (logit descending, index ascending):
//   w_i = exp((l_i - l_max) / T);  keep the first k;  of those the shortest prefix whose mass reaches p of theirs;
//   of those w_i >= min_p;  the token is the first (by index) whose running sum of kept weights exceeds u times their sum.
// T = 0 takes the first of the order.
//
// No row is sorted.  A cut of the ordered row is (key, m): everything above the key and the first m tokens equal to it.
// Keys are the logits' bits mapped to unsigned order; a cut is found by a radix selection on them, by counts for k, by
// mass for p.  Masses are 64-bit fixed point, w = W / 2^44: integer sums do not depend on the order in which atomics or
// CTAs add them, so the same row gives the same token on any launch, and W is computed in 64 bits, because an error of
// an fp32 exp moves all borders behind a likely token: over a large vocabulary u would meet a moved border once in a few
// hundred rows.
//
// A row belongs to a cluster of CTAs; each holds its slice of the keys in shared memory (the logits are read once), and
// the histograms and sums of the slices are read over distributed shared memory.  Bound by the chain of passes and
// cluster barriers when there are few rows, by the exponentials when there are many.
#pragma once

#include <cooperative_groups.h>

#include "ztq_common.cuh"

namespace ztq {

constexpr int kSampleThreads = 512;
constexpr int kSampleBins = 2048;                  // four per thread
constexpr int kSampleSeg = 256;                    // elements a warp takes at a time, eight per lane
constexpr int kSampleMaxCluster = 8;
constexpr int kSampleMaxSlice = 48640;             // keys of one CTA (fp32: 190 KB)
constexpr int kSampleMaxSegs = kSampleMaxSlice / kSampleSeg;
constexpr int kSampleFrac = 44;

struct SampleParams {
    const void* logits;
    long long stride;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int* token;
    float* logprob;
    int rows, vocab, slice, ranks, vec;
};

template <bool F32>
struct SampleKey;
template <>
struct SampleKey<true> {
    using T = uint32_t;
    static constexpr int kPasses = 3;
    static __device__ __forceinline__ int shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
    static __device__ __forceinline__ uint32_t mask(int pass) { return pass == 2 ? 1023u : 2047u; }
    static __device__ __forceinline__ uint32_t of(uint32_t u) {
        if ((u & 0x7fffffffu) > 0x7f800000u) return 0;         // NaN: below everything
        if (u == 0x80000000u) u = 0;                           // -0 is equal to 0
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        return k == 0 ? -__int_as_float(0x7f800000) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
    }
};
template <>
struct SampleKey<false> {
    using T = uint16_t;
    static constexpr int kPasses = 2;
    static __device__ __forceinline__ int shift(int pass) { return pass == 0 ? 5 : 0; }
    static __device__ __forceinline__ uint32_t mask(int pass) { return pass == 0 ? 2047u : 31u; }
    static __device__ __forceinline__ uint32_t of(uint32_t u) {
        if ((u & 0x7fffu) > 0x7c00u) return 0;
        if (u == 0x8000u) u = 0;
        return u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        return k == 0 ? -__int_as_float(0x7f800000) : h2f((uint16_t)(k & 0x8000u ? k & 0x7fffu : ~k));
    }
};

struct SampleShared {
    uint32_t hist[2][2][kSampleBins];              // [buffer][counts or low words of masses, high words][bin]
    unsigned long long seg_mass[kSampleMaxSegs];
    uint32_t seg_ties[kSampleMaxSegs];
    unsigned long long part[kSampleThreads / 32];
    unsigned long long mass;                       // read by the other ranks
    uint32_t ties, best;
    uint32_t found_bin;
    unsigned long long found_above, found_total;
};

// W of a logit
struct SampleWeight {
    double top, inv;
    bool top_inf;
    __device__ __forceinline__ unsigned long long operator()(float l) const {
        if (top_inf) return l > 3.402823466e38f ? 1ull << kSampleFrac : 0ull;
        const double x = ((double)l - top) * inv;
        if (!(x >= -31.2)) return 0ull;                        // also l = -inf times a vanishing 1/T
        return (unsigned long long)__double2ll_rn(exp(x) * (double)(1ull << kSampleFrac));
    }
};

template <typename V>
__device__ __forceinline__ V sample_warp_scan(V v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

template <bool F32>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
    namespace cg = cooperative_groups;
    using Key = SampleKey<F32>;
    using KT = typename Key::T;
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
    KT* keys = reinterpret_cast<KT*>(smem + ((sizeof(SampleShared) + 15) & ~15));
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = kSampleThreads / 32;
    const int ranks = p.ranks, rank = blockIdx.x % ranks, row = blockIdx.x / ranks;
    const int lo = min(rank * p.slice, p.vocab), n = min(p.slice, p.vocab - lo);
    const int segs = (n + kSampleSeg - 1) / kSampleSeg;

    grid_dep_launch();
    grid_dep_wait();
    // ---- the slice's keys and their largest
    uint32_t best = 0;
    for (int s = warp; s < segs; s += warps) {
        const int e = s * kSampleSeg;
        const long long at = row * p.stride + lo + e;
        if (p.vec && e + kSampleSeg <= n) {
            KT k[8];
            if constexpr (F32) {
                const uint4* g = reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(p.logits) + at + 8 * lane);
                const uint4 a = g[0], b = g[1];
                const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) { k[i] = Key::of(u[i]); best = max(best, (uint32_t)k[i]); }
                uint4* d = reinterpret_cast<uint4*>(keys + e + 8 * lane);
                d[0] = make_uint4(k[0], k[1], k[2], k[3]);
                d[1] = make_uint4(k[4], k[5], k[6], k[7]);
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.logits) + at + 8 * lane);
                const uint32_t u[4] = {a.x, a.y, a.z, a.w};
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t x = Key::of(u[i] & 0xffffu), y = Key::of(u[i] >> 16);
                    best = max(best, max(x, y));
                    w[i] = x | y << 16;
                }
                *reinterpret_cast<uint4*>(keys + e + 8 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = e + 32 * i + lane;
                uint32_t k = 0;
                if (j < n) {
                    if constexpr (F32) k = Key::of(static_cast<const uint32_t*>(p.logits)[row * p.stride + lo + j]);
                    else k = Key::of(static_cast<const uint16_t*>(p.logits)[row * p.stride + lo + j]);
                }
                keys[j] = (KT)k;                       // the padding of the last segment is key 0
                best = max(best, k);
            }
        }
    }
    best = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) sh.part[warp] = best;
    for (int i = tid; i < 2 * 2 * kSampleBins; i += kSampleThreads) (&sh.hist[0][0][0])[i] = 0;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < warps; ++w) best = max(best, (uint32_t)sh.part[w]);
        sh.best = best;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < ranks; ++r) best = max(best, *cluster.map_shared_rank(&sh.best, r));
    const float l_max = Key::value(best);

    // ---- the cut by temperature 0 or top-k: (cut, m)
    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    const int k = p.top_k && !greedy ? p.top_k[row] : 0;
    SampleWeight weight{(double)l_max, greedy ? 0.0 : 1.0 / (double)temp, l_max > 3.402823466e38f};
    uint32_t cut = 0;
    unsigned long long m = ~0ull >> 1;
    int buffer = 0;

    // The end of one pass of a radix selection: hist holds this rank's counts or masses by digit of the keys that share
    // the prefix found so far; the bin where the sum from the top (`above`: what lies above the prefix) reaches `want`
    // is found.  A negative `want` is a share of the whole and comes back as what it is worth.
    auto select = [&](double want, unsigned long long above, bool masses) {
        cluster.sync();                               // all ranks' histograms are complete
        unsigned long long mine[4] = {0, 0, 0, 0};
        for (int r = 0; r < ranks; ++r) {
            const uint4 a = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&sh.hist[buffer][0][4 * tid], r));
            mine[0] += a.x; mine[1] += a.y; mine[2] += a.z; mine[3] += a.w;
            if (masses) {
                const uint4 b = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&sh.hist[buffer][1][4 * tid], r));
                mine[0] += (unsigned long long)b.x << 32; mine[1] += (unsigned long long)b.y << 32;
                mine[2] += (unsigned long long)b.z << 32; mine[3] += (unsigned long long)b.w << 32;
            }
        }
        // thread t holds bins 4t .. 4t + 3
        const unsigned long long sum = mine[0] + mine[1] + mine[2] + mine[3];
        unsigned long long upto = sample_warp_scan(sum, lane);        // over lower threads of the warp, inclusive
        if (lane == 31) sh.part[warp] = upto;
        __syncthreads();
        unsigned long long total = 0, below = 0;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) below += sh.part[w];
            total += sh.part[w];
        }
        unsigned long long over = above + total - (below + upto);     // mass above this thread's bins
        if (want < 0) want = fmax(-want * (double)total, 0.5);        // a share of the whole (first pass of top-p)
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            if ((double)over < want && (double)(over + mine[i]) >= want) {
                sh.found_bin = 4 * tid + i;
                sh.found_above = over;
            }
            over += mine[i];
        }
        if (tid == 0) sh.found_total = total;
        // the other buffer was last read before the barrier above
        for (int i = tid; i < 2 * kSampleBins; i += kSampleThreads) (&sh.hist[buffer ^ 1][0][0])[i] = 0;
        buffer ^= 1;
        __syncthreads();
        return want;
    };

    if (best > Key::of(F32 ? 0xff800000u : 0xfc00u) && !greedy) {
        if (k > 0 && k < p.vocab) {
            uint32_t prefix = 0;
            unsigned long long above = 0;
            for (int pass = 0; pass < Key::kPasses; ++pass) {
                const int shift = Key::shift(pass);
                const uint32_t mask = Key::mask(pass);
                for (int s = warp; s < segs; s += warps)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t key = keys[s * kSampleSeg + 32 * i + lane];
                        if (pass == 0 || (key >> shift) >> (pass == 1 ? (F32 ? 11 : 5) : 10) == prefix) atomicAdd(&sh.hist[buffer][0][(key >> shift) & mask], 1u);
                    }
                select((double)k, above, false);
                above = sh.found_above;
                prefix = prefix << (pass == 0 ? 0 : pass == 1 ? (F32 ? 11 : 5) : 10) | sh.found_bin;
            }
            cut = prefix;
            m = (unsigned long long)k - above;
        }
        // ---- the cut by top-p, among what top-k left
        const float share = p.top_p ? p.top_p[row] : 1.f;
        if (share < 1.f) {
            const unsigned long long tie = cut ? weight(Key::value(cut)) : 0ull;
            uint32_t prefix = 0;
            unsigned long long above = 0;
            double want = -(double)fmaxf(share, 0.f);
            if (want == 0.0) want = 0.5;               // nothing wanted: the first token alone
            for (int pass = 0; pass < Key::kPasses; ++pass) {
                const int shift = Key::shift(pass), up = pass == 0 ? 0 : pass == 1 ? (F32 ? 11 : 5) : 10;
                const uint32_t mask = Key::mask(pass);
                auto add = [&](uint32_t key, unsigned long long w) {
                    const uint32_t bin = (key >> shift) & mask, low = (uint32_t)w;
                    const uint32_t old = low ? atomicAdd(&sh.hist[buffer][0][bin], low) : 0u;
                    const uint32_t high = (uint32_t)(w >> 32) + (low && old + low < low);
                    if (high) atomicAdd(&sh.hist[buffer][1][bin], high);
                };
                for (int s = warp; s < segs; s += warps)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t key = keys[s * kSampleSeg + 32 * i + lane];
                        if (key > cut && (pass == 0 || (key >> shift) >> up == prefix)) {
                            const unsigned long long w = weight(Key::value(key));
                            if (w) add(key, w);
                        }
                    }
                if (tie && rank == 0 && tid == 0 && (pass == 0 || (cut >> shift) >> up == prefix)) add(cut, m * tie);
                want = select(want, above, true);
                above = sh.found_above;
                prefix = prefix << up | sh.found_bin;
            }
            cut = prefix;
            const unsigned long long w = weight(Key::value(cut));
            m = (unsigned long long)ceil((want - (double)above) / (double)w);
            if (m < 1) m = 1;
        }
    }
    if (greedy) { cut = best; m = 1; }

    // ---- sums of what is kept, by segments in the order of the vocabulary
    const float floor_p = p.min_p && !greedy && p.min_p[row] > 0.f ? fminf(p.min_p[row], 1.f) : 0.f;
    const double l_min = floor_p > 0.f ? (double)l_max + (double)temp * log((double)floor_p) : -1e300;
    const bool tie_kept = (double)Key::value(cut) >= l_min;
    const unsigned long long tie = !tie_kept ? 0ull : greedy ? 1ull : weight(Key::value(cut));
    auto strict = [&](uint32_t key) {                  // weight of a key above the cut
        const float l = Key::value(key);
        return key > cut && (double)l >= l_min ? weight(l) : 0ull;
    };
    for (int s = warp; s < segs; s += warps) {
        unsigned long long w = 0;
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t key = keys[s * kSampleSeg + 32 * i + lane];
            if (key > cut) w += strict(key);
            c += key == cut;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) { sh.seg_mass[s] = w; sh.seg_ties[s] = c; }
    }
    __syncthreads();
    if (warp == 0) {
        unsigned long long w = 0;
        uint32_t c = 0;
        for (int s = lane; s < segs; s += 32) { w += sh.seg_mass[s]; c += sh.seg_ties[s]; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) { sh.mass = w; sh.ties = c; }
    }
    cluster.sync();
    unsigned long long total = 0, before = 0, ties_before = 0, mine = 0, ties = 0;
    for (int r = 0; r < ranks; ++r) {
        const unsigned long long c = *cluster.map_shared_rank(&sh.ties, r);
        const unsigned long long kept = m > ties ? min(c, m - ties) : 0ull;
        const unsigned long long w = *cluster.map_shared_rank(&sh.mass, r) + kept * tie;
        if (r == rank) { before = total; ties_before = ties; mine = w; }
        total += w;
        ties += c;
    }
    cluster.sync();                                    // nobody's shared memory is read after this
    if (total == 0) {                                  // no finite logit (or none but NaN)
        if (rank == 0 && tid == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = __int_as_float(0x7fc00000);
        }
        return;
    }
    const float u = p.uniform ? p.uniform[row] : 0.f;
    const double u01 = u > 0.f ? fmin((double)u, 1.0 - 1.0 / 16777216) : 0.0;
    const unsigned long long target = min((unsigned long long)(u01 * (double)total), total - 1);
    if (warp != 0 || target < before || target >= before + mine) return;
    // ---- this CTA holds the token: its segment, then the element
    unsigned long long at = before, t_at = ties_before;
    int seg = -1;
    for (int s0 = 0; s0 < segs && seg < 0; s0 += 32) {
        const int s = s0 + lane;
        const unsigned long long c = s < segs ? sh.seg_ties[s] : 0ull;
        const unsigned long long c_upto = t_at + sample_warp_scan(c, lane), c_before = c_upto - c;
        const unsigned long long w = (s < segs ? sh.seg_mass[s] : 0ull) + (m > c_before ? min(c, m - c_before) : 0ull) * tie;
        const unsigned long long upto = at + sample_warp_scan(w, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, upto > target);
        const int src = hit ? __ffs(hit) - 1 : 31;
        const unsigned long long w_src = __shfl_sync(0xffffffffu, upto - (hit ? w : 0ull), src);
        const unsigned long long t_src = __shfl_sync(0xffffffffu, hit ? c_before : c_upto, src);
        at = w_src;
        t_at = t_src;
        if (hit) seg = s0 + src;
    }
    for (int i = 0; i < 8; ++i) {
        const int j = seg * kSampleSeg + 32 * i + lane;
        const uint32_t key = keys[j];
        const bool is_tie = key == cut;
        const unsigned eq = __ballot_sync(0xffffffffu, is_tie);
        const unsigned long long c_before = t_at + __popc(eq & ((1u << lane) - 1));
        const unsigned long long w = is_tie ? (c_before < m ? tie : 0ull) : key > cut ? strict(key) : 0ull;
        const unsigned long long upto = at + sample_warp_scan(w, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, upto > target);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                p.token[row] = lo + j;
                if (p.logprob)
                    p.logprob[row] = greedy ? 0.f : (float)((weight.top_inf ? 0.0 : ((double)Key::value(key) - weight.top) * weight.inv) -
                                                            log((double)total / (double)(1ull << kSampleFrac)));
            }
            return;
        }
        at = __shfl_sync(0xffffffffu, upto, 31);
        t_at += __popc(eq);
    }
}

}  // namespace ztq
