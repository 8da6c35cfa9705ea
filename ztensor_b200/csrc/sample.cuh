// sample.cuh -- one token per row of logits, from a given random number.
//
// With l_max the largest logit, T the temperature and the tokens ordered by (logit descending, index ascending):
//   w_i = exp((l_i - l_max) / T);  keep the first k;  of those the shortest prefix whose mass reaches p of theirs;
//   of those w_i >= min_p;  the token is the first (by index) whose running sum of kept weights exceeds u times their sum.
// T = 0 takes the first of the order.
//
// No row is sorted.  A cut of the ordered row is (key, m): everything above the key and the first m tokens equal to it.
// Keys are the logits' bits mapped to unsigned order.  A cut is found in steps, by counts for k and by mass for p: a
// histogram over log2(w) in 16ths (on the bits of the logits most of a row would fall into a few dozen bins, whose atomics
// serialize), if its bin holds more than a few keys a second one over 1024ths of that bin, then the keys that are left
// compared with one another; where they are still more than 511 (ties, or a bin without a lower end), a radix selection.
// Masses are 64-bit fixed point, w = W / 2^44: integer sums do not depend on the order in which atomics or CTAs add them, so
// the same row gives the same token on any launch, and W is computed in 64 bits, because an error of an fp32 exp moves all
// borders behind a likely token: over a large vocabulary u would meet a moved border once in a few hundred rows.
//
// Most rows are done earlier: the k-th largest of the maxima of groups of lanes is a lower bound of the k-th largest logit,
// min-p gives one directly.  Where at most kSampleList tokens reach the bound, one CTA takes them with their indices and
// ranks, sums and draws by comparing all pairs.
// Without top-k a token lighter than (1 - p) / vocab cannot end the nucleus (all lighter ones together weigh less than the
// share that top-p leaves out), so only heavier ones enter the histogram.
//
// A row belongs to a cluster of CTAs; each holds its slice of the keys in shared memory (the logits are read once), and
// the histograms and sums of the slices are read over distributed shared memory.  Bound by the chain of passes and
// cluster barriers when there are few rows, by the passes over the keys when there are many.  64 rows of 131072 fp16 logits:
// greedy 18 us, top-k 50 27, top-k 1000 48, min-p 24, top-p 0.9 alone 105; one row of 32000: 7, 11, 18, 9, 29.
#pragma once

#include <cooperative_groups.h>

#include <type_traits>

#include "ztq_common.cuh"

namespace ztq {

constexpr int kSampleThreads = 512;
constexpr int kSampleBins = 1024;                  // two per thread
constexpr int kSampleSeg = 256;                    // elements a warp takes at a time, eight per lane
constexpr int kSampleMaxCluster = 8;
constexpr int kSampleMaxSlice = 40960;             // keys of one CTA (fp32: 160 KB)
constexpr int kSampleMaxSegs = kSampleMaxSlice / kSampleSeg;
constexpr int kSampleFrac = 44;
constexpr int kSampleCand = kSampleThreads;        // keys of a bin that are compared directly, of all ranks
constexpr int kSampleFew = 64;                     // below this they are compared at once, else the bin is divided further first
constexpr int kSampleList = 192;                   // tokens that are ranked directly
constexpr int kSampleKeep = 2048;                  // keys of a slice that are kept apart, so that later passes need not look at all
constexpr int kSampleGroups = 4;                   // groups of lanes of a warp whose maxima are kept

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
    static constexpr int kPasses = 4;                  // digits of a radix selection
    static __device__ __forceinline__ int shift(int pass) { return pass < 3 ? 22 - 10 * pass : 0; }
    static __device__ __forceinline__ int bits(int pass) { return pass < 3 ? 10 : 2; }
    static __device__ __forceinline__ uint32_t of(uint32_t u) {
        if ((u & 0x7fffffffu) > 0x7f800000u) return 0;         // NaN: below everything
        if (u == 0x80000000u) u = 0;                           // -0 is equal to 0
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        return k == 0 ? -__int_as_float(0x7f800000) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
    }
    static __device__ __forceinline__ uint32_t least(double v) { return of(__float_as_uint(__double2float_ru(v))); }   // of the values >= v
};
template <>
struct SampleKey<false> {
    using T = uint16_t;
    static constexpr int kPasses = 2;
    static __device__ __forceinline__ int shift(int pass) { return pass == 0 ? 6 : 0; }
    static __device__ __forceinline__ int bits(int pass) { return pass == 0 ? 10 : 6; }
    static __device__ __forceinline__ uint32_t of(uint32_t u) {
        if ((u & 0x7fffu) > 0x7c00u) return 0;
        if (u == 0x8000u) u = 0;
        return u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        return k == 0 ? -__int_as_float(0x7f800000) : h2f((uint16_t)(k & 0x8000u ? k & 0x7fffu : ~k));
    }
    static __device__ __forceinline__ uint32_t least(double v) { return of(__half_as_ushort(__float2half_ru(__double2float_ru(v)))); }
};

struct SampleShared {
    uint32_t hist[2][3][kSampleBins];              // [buffer][counts, or the 16-bit digits of masses][bin]: a slice's digits add up below 2^32
    unsigned long long seg_mass[kSampleMaxSegs];
    uint32_t seg_ties[kSampleMaxSegs];
    unsigned long long part[kSampleThreads / 32];
    unsigned long long mass;                       // read by the other ranks
    uint32_t ties, best, group_best[kSampleThreads / 32 * kSampleGroups], warp_low[kSampleThreads / 32], low;
    uint32_t index[kSampleCand];                   // of the tokens in cand
    uint32_t found_bin, cands, found_key;
    uint32_t cand[kSampleCand], all[kSampleCand];
    unsigned long long all_mass[kSampleCand];
    uint32_t list[kSampleKeep];
    unsigned long long found_above, found_total;
};

// 2^x 2^44 for x in [-46, 0], rounded: 2^n by the exponent, 2^f for |f| <= 1/2 by the Taylor series of exp(f ln 2), whose
// first omitted term is (ln 2 / 2)^12 / 12! < 2^-47.
__device__ __forceinline__ unsigned long long sample_exp2(double x) {
    const double big = 6755399441055744.0, t = x + big, f = x - (t - big);      // 1.5 2^52: the sum ends in the nearest integer
    const int n = __double2loint(t);
    double y = 4.4455382718708116e-10;                             // ln2^11 / 11!, and so on down
    y = fma(y, f, 7.0549116208011234e-09);
    y = fma(y, f, 1.0178086009239700e-07);
    y = fma(y, f, 1.3215486790144309e-06);
    y = fma(y, f, 1.5252733804059841e-05);
    y = fma(y, f, 1.5403530393381609e-04);
    y = fma(y, f, 1.3333558146428443e-03);
    y = fma(y, f, 9.6181291076284772e-03);
    y = fma(y, f, 5.5504108664821580e-02);
    y = fma(y, f, 2.4022650695910071e-01);
    y = fma(y, f, 6.9314718055994531e-01);
    y = fma(y, f, 1.0);
    y = __hiloint2double(__double2hiint(y) + ((n + kSampleFrac) << 20), __double2loint(y)) + 4503599627370496.0;      // 2^52: ends in the integer
    return (unsigned long long)__double_as_longlong(y) & 0xfffffffffffffull;
}

// W of a logit
struct SampleWeight {
    double top, c;                                                 // c: log2(e) / T
    bool top_inf;
    __device__ __forceinline__ unsigned long long operator()(float l) const {
        if (top_inf) return l > 3.402823466e38f ? 1ull << kSampleFrac : 0ull;
        const double x = ((double)l - top) * c;
        if (!(x >= -45.0)) return 0ull;                            // also l = -inf times a vanishing 1/T
        return sample_exp2(x);
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
    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    int k = p.top_k && !greedy ? p.top_k[row] : 0;
    if (greedy) k = 1;
    if (k >= p.vocab) k = 0;
    const float share = p.top_p && !greedy ? p.top_p[row] : 1.f;
    const float floor_p = p.min_p && !greedy && p.min_p[row] > 0.f ? fminf(p.min_p[row], 1.f) : 0.f;
    // ---- the slice's keys and their largest
    uint32_t best = 0;
    // The logits come as they are, all copies in flight at once; each lane then turns what it copied itself into keys.
    // Pieces of 16 bytes where rows are aligned, single floats else, halves of unaligned rows through registers.
    constexpr int kPer = 16 / sizeof(KT);                  // keys of a piece
    const KT* row_at = static_cast<const KT*>(p.logits) + row * p.stride + lo;
    for (int s = warp; s < segs; s += warps) {
        const int e = s * kSampleSeg;
        if (p.vec && e + kSampleSeg <= n) {
#pragma unroll
            for (int i = 0; i < 8 / kPer; ++i) {
                const int j = e + (32 * i + lane) * kPer;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(keys + j)), "l"(row_at + j) : "memory");
            }
        } else if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = e + 32 * i + lane;
                if (j < n) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(keys + j)), "l"(row_at + j) : "memory");
            }
        } else {
            KT v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = e + 32 * i + lane;
                v[i] = j < n ? row_at[j] : 0;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) keys[e + 32 * i + lane] = v[i];
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int s = warp; s < segs; s += warps) {
        const int e = s * kSampleSeg;
        if (p.vec && e + kSampleSeg <= n) {
#pragma unroll
            for (int i = 0; i < 8 / kPer; ++i) {
                uint4* at = reinterpret_cast<uint4*>(keys + e + (32 * i + lane) * kPer);
                uint4 v = *at;
                uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                for (int k4 = 0; k4 < 4; ++k4) {
                    if constexpr (F32) {
                        w[k4] = Key::of(w[k4]);
                        best = max(best, w[k4]);
                    } else {
                        const uint32_t x = Key::of(w[k4] & 0xffffu), y = Key::of(w[k4] >> 16);
                        best = max(best, max(x, y));
                        w[k4] = x | y << 16;
                    }
                }
                *at = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = e + 32 * i + lane;
                const uint32_t key = j < n ? Key::of(keys[j]) : 0;         // the padding of the last segment is key 0
                keys[j] = (KT)key;
                best = max(best, key);
            }
        }
    }
    // maxima of groups of lanes for a bound of the k-th largest; with too many wanted for that, the q-th largest lane of
    // every warp, whose least over all warps is one too
    const int groups = ranks * warps * kSampleGroups, quota = k > 0 && 2 * k > groups ? (k + ranks * warps - 1) / (ranks * warps) : 0;
    uint32_t group = best, low = 0;
#pragma unroll
    for (int o = 1; o < 32 / kSampleGroups; o <<= 1) group = max(group, __shfl_xor_sync(0xffffffffu, group, o));
    if (lane % (32 / kSampleGroups) == 0) sh.group_best[warp * kSampleGroups + lane / (32 / kSampleGroups)] = group;
    if (quota > 0 && quota <= 32) {
        uint32_t left = best;
        for (int i = 0; i < quota; ++i) {
            low = __reduce_max_sync(0xffffffffu, left);
            const unsigned who = __ballot_sync(0xffffffffu, left == low);
            if (lane == __ffs(who) - 1) left = 0;
        }
    }
    best = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) { sh.part[warp] = best; sh.warp_low[warp] = low; }
    if (tid == 0) sh.cands = 0;
    for (int i = tid; i < 2 * 3 * kSampleBins; i += kSampleThreads) (&sh.hist[0][0][0])[i] = 0;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < warps; ++w) {
            best = max(best, (uint32_t)sh.part[w]);
            low = min(low, sh.warp_low[w]);
        }
        sh.best = best;
        sh.low = low;
    }
    cluster.sync();
    best = 0;
    low = 0xffffffffu;
    for (int r = 0; r < ranks; ++r) {
        best = max(best, *cluster.map_shared_rank(&sh.best, r));
        low = min(low, *cluster.map_shared_rank(&sh.low, r));
    }
    const float l_max = Key::value(best);

    const SampleWeight weight{(double)l_max, greedy ? 0.0 : 1.4426950408889634 / (double)temp, l_max > 3.402823466e38f};
    // a logit's place in the histogram: the distance to the largest in 16ths of log2(w), largest last
    const float c16 = greedy ? 0.f : 16.f * 1.44269504f / temp;
    auto coarse = [&](float l) {
        const float d = (l_max - l) * c16;
        return l == l_max ? kSampleBins - 1 : d < (float)(kSampleBins - 1) ? kSampleBins - 1 - (int)d : 0;
    };
    auto fine = [&](float l) {                             // its place within a bin other than 0
        const float d = l == l_max ? 0.f : (l_max - l) * c16;
        return kSampleBins - 1 - (int)((d - floorf(d)) * (float)kSampleBins);
    };
    const double l_min = floor_p > 0.f ? (double)l_max + (double)temp * log((double)floor_p) : -1e300;
    const uint32_t key_min = floor_p > 0.f ? Key::least(l_min) : 0;
    const bool any = best > Key::of(F32 ? 0xff800000u : 0xfc00u);         // something to draw
    // ---- a bound below which nothing is kept
    if (greedy) low = best;
    else if (k > 0 && 2 * k <= groups) {
        // the k-th largest of the groups' maxima; of the warps' where they are enough
        const int step = 2 * k <= ranks * warps ? kSampleGroups : 1, n_g = groups / step;
        for (int i = tid; i < n_g; i += kSampleThreads) {
            const int per = warps * kSampleGroups / step;
            const uint32_t* from = cluster.map_shared_rank(&sh.group_best[0], i / per) + i % per * step;
            uint32_t v = from[0];
            for (int j = 1; j < step; ++j) v = max(v, from[j]);
            sh.all[i] = v;
        }
        __syncthreads();
        if (tid < n_g) {
            const uint32_t v = sh.all[tid];
            int over = 0;
#pragma unroll 8
            for (int j = 0; j < n_g; ++j) over += sh.all[j] > v || (sh.all[j] == v && j < tid);
            if (over == k - 1) sh.found_key = v;
        }
        __syncthreads();
        low = sh.found_key;
    } else if (k <= 0) low = key_min;
    // f(key) for the slice's keys
    auto each = [&](auto f) {
        for (int s = warp; s < segs; s += warps)
#pragma unroll
            for (int i = 0; i < 8; ++i) f((uint32_t)keys[s * kSampleSeg + 32 * i + lane]);
    };
    // f(key, logit, weight) for the keys of segment s; the weight is 0 where test(key) is false
    auto each_weight = [&](int s, auto test, auto f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t key = keys[s * kSampleSeg + 32 * i + lane];
            const float l = Key::value(key);
            f(key, l, test(key) ? weight(l) : 0ull);
        }
    };
    const float u = p.uniform ? p.uniform[row] : 0.f;
    const double u01 = u > 0.f ? fmin((double)u, 1.0 - 1.0 / 16777216) : 0.0;
    auto say = [&](int token, float l, unsigned long long total) {
        p.token[row] = token;
        if (p.logprob)
            p.logprob[row] = greedy ? 0.f : (float)((weight.top_inf ? 0.0 : ((double)l - weight.top) / (double)temp) - log((double)total / (double)(1ull << kSampleFrac)));
    };

    int n_list = -1;                                       // keys in sh.list, if they are all that matters
    // ---- few tokens reach the bound: rank 0 takes them all
    if (any && low > 0) {
        const bool whole = k <= 0 && share < 1.f;          // top-p of everything: its mass is wanted too
        unsigned long long sum = 0;
        for (int s = warp; s < segs; s += warps) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = s * kSampleSeg + 32 * i + lane;
                const uint32_t key = keys[j];
                if (key >= low) {
                    const uint32_t at = atomicAdd(&sh.cands, 1u);
                    if (at < kSampleList) { sh.cand[at] = key; sh.index[at] = (uint32_t)(lo + j); }
                    if (at < kSampleKeep) sh.list[at] = key;
                }
            }
            if (whole) each_weight(s, [](uint32_t) { return true; }, [&](uint32_t, float, unsigned long long w) { sum += w; });
        }
        if (whole) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sh.part[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < warps; ++w) sum += sh.part[w];
                sh.mass = sum;
            }
        }
        cluster.sync();
        int n_l = 0;
        for (int r = 0; r < ranks; ++r) n_l += (int)min(*cluster.map_shared_rank(&sh.cands, r), (uint32_t)kSampleList + 1);
        if (n_l <= kSampleList) {
            if (rank == 0) {
                // entries {order: key, then the lower index first; mass}, read whole by every thread
                ulonglong2* entry = reinterpret_cast<ulonglong2*>(&sh.hist[0][0][0]);       // not needed any more
                unsigned long long z = 0;
                int at = 0;
                unsigned long long order = 0, w = 0;
                uint32_t key = 0, id = 0;
                for (int r = 0; r < ranks; ++r) {
                    const int c = (int)*cluster.map_shared_rank(&sh.cands, r);
                    if (tid >= at && tid < at + c) {
                        key = cluster.map_shared_rank(&sh.cand[0], r)[tid - at];
                        id = cluster.map_shared_rank(&sh.index[0], r)[tid - at];
                    }
                    if (whole) z += *cluster.map_shared_rank(&sh.mass, r);
                    at += c;
                }
                const bool has = tid < n_l;
                if (has) {
                    order = (unsigned long long)key << 32 | (0xffffffffu - id);
                    w = weight(Key::value(key));
                    entry[tid] = make_ulonglong2(order, w);
                }
                __syncthreads();
                int place = 0;
                unsigned long long ahead = 0;
                if (has)
#pragma unroll 8
                    for (int j = 0; j < n_l; ++j) {
                        const ulonglong2 o = entry[j];
                        if (o.x > order) { ++place; ahead += o.y; }
                    }
                // what stands ahead of a token that top-k keeps is kept as well; the last such token has the sum of all
                const bool kept_k = has && (k <= 0 || place < k);
                if (kept_k && place == (k > 0 ? min(k, n_l) : n_l) - 1) sh.found_total = ahead + w;
                __syncthreads();
                const double wanted = (double)share * (double)(whole ? z : sh.found_total);
                const bool kept = kept_k && key >= key_min && (share >= 1.f || place == 0 || (double)ahead < wanted);
                if (has) entry[tid] = make_ulonglong2((unsigned long long)id, kept ? w : 0ull);
                __syncthreads();
                unsigned long long before = 0, total = 0;
                if (has)
#pragma unroll 8
                    for (int j = 0; j < n_l; ++j) {
                        const ulonglong2 o = entry[j];
                        total += o.y;
                        if (o.x < id) before += o.y;
                    }
                const unsigned long long target = total ? min((unsigned long long)(u01 * (double)total), total - 1) : 0;
                if (kept && w && before <= target && target < before + w) say((int)id, Key::value(key), total);
            }
            cluster.sync();                                // the lists have been read
            return;
        }
        if (k > 0 && sh.cands <= kSampleKeep) n_list = (int)sh.cands;
        cluster.sync();                                    // the counters and sums have been read
    }

    uint32_t cut = 0;
    unsigned long long m = ~0ull >> 1;
    int buffer = 0;

    // The end of one pass of a radix selection: hist holds this rank's counts or masses by digit of the keys that share
    // the prefix found so far; the bin where the sum from the top (`above`: what lies above the prefix) reaches `want`
    // is found.  A negative `want` is a share of the whole and comes back as what it is worth.
    auto select = [&](double want, unsigned long long above, bool masses) {
        cluster.sync();                               // all ranks' histograms are complete
        unsigned long long mine[2] = {0, 0};           // thread t holds bins 2t and 2t + 1
        for (int r = 0; r < ranks; ++r) {
#pragma unroll
            for (int d = 0; d < 3; ++d) {
                if (d && !masses) break;
                const uint2 a = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&sh.hist[buffer][d][2 * tid], r));
                mine[0] += (unsigned long long)a.x << 16 * d;
                mine[1] += (unsigned long long)a.y << 16 * d;
            }
        }
        const unsigned long long sum = mine[0] + mine[1];
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
        for (int i = 1; i >= 0; --i) {
            if ((double)over < want && (double)(over + mine[i]) >= want) {
                sh.found_bin = 2 * tid + i;
                sh.found_above = over;
            }
            over += mine[i];
        }
        if (tid == 0) sh.found_total = total;
        // the other buffer was last read before the barrier above
        for (int i = tid; i < 3 * kSampleBins; i += kSampleThreads) (&sh.hist[buffer ^ 1][0][0])[i] = 0;
        buffer ^= 1;
        __syncthreads();
        return want;
    };

    auto add_mass = [&](uint32_t bin, unsigned long long w) {
        const uint32_t d0 = (uint32_t)w & 0xffffu, d1 = (uint32_t)w >> 16, d2 = (uint32_t)(w >> 32);
        if (d0) atomicAdd(&sh.hist[buffer][0][bin], d0);
        if (d1) atomicAdd(&sh.hist[buffer][1][bin], d1);
        if (d2) atomicAdd(&sh.hist[buffer][2][bin], d2);
    };
    // The cut where counts (MASSES: masses) of the keys above `floor`, and of `floor` itself as one of `floor_mass`, summed
    // from the top reach `want`; it is not below `least`.  Leaves the sum above the cut in sh.found_above.
    auto find = [&](double& want, uint32_t floor, unsigned long long floor_mass, uint32_t least, auto masses) -> uint32_t {
        constexpr bool MASSES = decltype(masses)::value;
        const bool first = rank == 0 && tid == 0 && floor_mass != 0;      // the one who adds the floor's mass
        unsigned long long rest = 0;
        int kept = n_list;                                // keys of sh.list to go through instead of all; -1: all
        auto each_kept = [&](auto f) {
            if (kept < 0) each(f);
            else for (int i = tid; i < kept; i += kSampleThreads) f(sh.list[i]);
        };
        each_kept([&](uint32_t key) {
            if constexpr (MASSES) {
                if (key <= floor) return;
                const float l = Key::value(key);
                const unsigned long long w = weight(l);
                if (key < least) rest += w;
                else if (w) add_mass(coarse(l), w);
            } else if (key >= least) atomicAdd(&sh.hist[buffer][0][coarse(Key::value(key))], 1u);
        });
        if constexpr (MASSES) {                           // (its high digit takes part of 32 bits: at most 16 such adds)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
            if (lane == 0 && rest) add_mass(0, rest);
        }
        if (first) add_mass(coarse(Key::value(floor)), floor_mass);
        if (tid == 0) sh.cands = 0;
        want = select(want, 0, MASSES);
        unsigned long long above = sh.found_above;
        const int bin = (int)sh.found_bin;
        // keys of the bin; of one 1024th of it in the second round
        int fine_bin = -1;
        auto inside = [&](uint32_t key) {
            if (key < least || (key <= floor && floor)) return false;
            const float l = Key::value(key);
            return coarse(l) == bin && (fine_bin < 0 || fine(l) == fine_bin);
        };
        auto floor_inside = [&]() {
            const float l = Key::value(floor);
            return floor_mass != 0 && coarse(l) == bin && (fine_bin < 0 || fine(l) == fine_bin);
        };
        for (int round = 0;; ++round) {
            const bool fills = kept < 0;                      // the list is free: it takes the bin's keys
            each_kept([&](uint32_t key) {
                if (inside(key)) {
                    const uint32_t at = atomicAdd(&sh.cands, 1u);
                    if (at < kSampleCand) sh.cand[at] = key;
                    if (fills && at < kSampleKeep) sh.list[at] = key;
                }
            });
            cluster.sync();
            if (fills && sh.cands <= kSampleKeep) kept = (int)sh.cands;
            uint32_t total = 0;
            for (int r = 0; r < ranks; ++r) total += min(*cluster.map_shared_rank(&sh.cands, r), (uint32_t)kSampleCand);
            if (total < (round ? kSampleCand : kSampleFew)) {
                uint32_t at = 0;
                for (int r = 0; r < ranks; ++r) {
                    const uint32_t c = *cluster.map_shared_rank(&sh.cands, r);
                    if (tid >= at && tid < at + c) sh.all[tid] = cluster.map_shared_rank(&sh.cand[0], r)[tid - at];
                    at += c;
                }
                const bool with_floor = floor_inside();
                if (with_floor && tid == total) sh.all[total] = floor;
                if (with_floor) ++total;
                __syncthreads();
                uint32_t key = 0;
                if (tid < total) {
                    key = sh.all[tid];
                    if constexpr (MASSES) sh.all_mass[tid] = with_floor && tid == total - 1 ? floor_mass : weight(Key::value(key));
                }
                __syncthreads();
                if (tid < total) {
                    unsigned long long over = above, same = 0;
#pragma unroll 8
                    for (uint32_t j = 0; j < total; ++j) {
                        const uint32_t other = sh.all[j];
                        const unsigned long long w = MASSES ? sh.all_mass[j] : 1ull;
                        if (other > key) over += w;
                        if (other == key) same += w;
                    }
                    if ((double)over < want && (double)(over + same) >= want) {
                        sh.found_key = key;
                        sh.found_above = over;
                    }
                }
                cluster.sync();                               // the lists have been read, the cut is there
                return sh.found_key;
            }
            cluster.sync();                                   // the counters have been read
            if (round == 1 || bin == 0) break;                // bin 0 has no lower end
            if (tid == 0) sh.cands = 0;
            each_kept([&](uint32_t key) {
                if (!inside(key)) return;
                const float l = Key::value(key);
                if constexpr (MASSES) {
                    const unsigned long long w = weight(l);
                    if (w) add_mass(fine(l), w);
                } else atomicAdd(&sh.hist[buffer][0][fine(l)], 1u);
            });
            if (first && floor_inside()) add_mass(fine(Key::value(floor)), floor_mass);
            select(want, above, MASSES);
            above = sh.found_above;
            fine_bin = (int)sh.found_bin;
        }
        const bool with_floor = floor_inside();
        uint32_t prefix = 0;
        for (int pass = 0; pass < Key::kPasses; ++pass) {
            const int shift = Key::shift(pass), up = Key::bits(pass);
            const uint32_t mask = (1u << up) - 1;
            auto matches = [&](uint32_t key) { return pass == 0 || (key >> shift) >> up == prefix; };
            each_kept([&](uint32_t key) {
                if (!inside(key) || !matches(key)) return;
                if constexpr (MASSES) {
                    const unsigned long long w = weight(Key::value(key));
                    if (w) add_mass((key >> shift) & mask, w);
                } else atomicAdd(&sh.hist[buffer][0][(key >> shift) & mask], 1u);
            });
            if (first && with_floor && matches(floor)) add_mass((floor >> shift) & mask, floor_mass);
            select(want, above, MASSES);
            above = sh.found_above;
            prefix = prefix << up | sh.found_bin;
        }
        return prefix;
    };

    if (any && !greedy) {
        if (k > 0) {
            double want = (double)k;
            cut = find(want, 0, 0, low, std::false_type());
            m = (unsigned long long)k - sh.found_above;
        }
        // ---- the cut by top-p, among what top-k left
        if (share < 1.f) {
            double want = share > 0.f ? -(double)share : 0.5;          // nothing wanted: the first token alone
            const unsigned long long tie = cut ? weight(Key::value(cut)) : 0ull;
            // half of (1 - p) / vocab: room for the rounding of the bound itself
            const double light = 0.5 * (1.0 - fmax((double)share, 0.0)) / p.vocab;
            cut = find(want, cut, m * tie, k > 0 ? 0u : Key::least((double)l_max + (double)temp * log(light)), std::true_type());
            const unsigned long long w = weight(Key::value(cut));
            m = (unsigned long long)ceil((want - (double)sh.found_above) / (double)w);
            if (m < 1) m = 1;
        }
    }
    if (greedy) { cut = best; m = 1; }

    // ---- sums of what is kept, by segments in the order of the vocabulary
    const unsigned long long tie = !any || cut < key_min ? 0ull : greedy ? 1ull : weight(Key::value(cut));
    auto strict = [&](uint32_t key) { return key > cut && key >= key_min ? weight(Key::value(key)) : 0ull; };     // of a key above the cut
    for (int s = warp; s < segs; s += warps) {
        unsigned long long w = 0;
        uint32_t c = 0;
        each_weight(s, [&](uint32_t key) { return key > cut && key >= key_min; }, [&](uint32_t key, float, unsigned long long x) {
            w += x;
            c += key == cut;
        });
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
            if (lane == __ffs(hit) - 1) say(lo + j, Key::value(key), total);
            return;
        }
        at = __shfl_sync(0xffffffffu, upto, 31);
        t_at += __popc(eq);
    }
}

}  // namespace ztq
