// rope_append.cuh -- rotary positions, and the append of a step's keys and values to the paged 8-bit cache.
//
// Rotation of a pair (a, b) at position m with frequency f_i:
//   (a cos - b sin, b cos + a sin),  cos and sin of m f_i from a table [positions][rot / 2] of fp32 {cos, sin}; the
// table is made once, in 64 bits (a far position times a frequency loses its angle in 32).  Halves: (i, i + rot/2);
// pairs: (2i, 2i + 1).  Arithmetic in fp32, one rounding to fp16 where the output is fp16.
//
// The cache holds int8 codes with one scale per (block, head), keys and values apart.  When rows are added to a block
//   need  = the smallest power of two with max|new rows| <= 127 need
//   scale' = max(scale, need)            (need alone when the first new row is the block's first)
//   old codes = rint(code scale / scale'), new codes = rint(x / scale').
// A power of two makes x / scale' exact, so the only rounding is the one to a code (half a step), and growth costs the
// old rows at most the half step they are entitled to at the new scale.  A non-finite new row makes the scale NaN.
//
// Work: units of 16 elements of one head.  A CTA holds a tile of kTokenTile rows, for a group of query heads or for the
// keys or values of one head.  Queries: a thread keeps one (row, unit) and its eight cosines and sines and goes through the heads.
// The rows of one block stand together (a run); the CTA whose tile holds a run's first row does the whole run, so a block
// has one writer and needs no atomics.  Keys and values are two CTAs.  With few runs in the tile (a prompt) the whole CTA
// takes each run, with many (decoding) every warp takes runs of its own.  The rows are read twice, for the largest value
// and for the rounding; the second time they come from L1 (holding them in registers cost the queries' part its occupancy).
// 8192 rows, 32 + 8 + 8 heads of 128 in fp16 (186 MB, 29 us of HBM time) take 60 us, the queries alone 35: the chain slots ->
// rows -> scale -> rows again of 2048 CTAs is not hidden behind the copies.  Eight decoding rows: 4 us, the chain once.
#pragma once

#include "ztq_common.cuh"

namespace ztq {

constexpr int kRopeThreads = 256;
constexpr int kTokenTile = 16;                     // rows of a tile of queries
constexpr int kMaxKvTile = 64;                     // of keys and values: 64 for many rows, where most tiles of 16 would begin no run

struct RopeParams {
    const float2* table;       // [table_rows][half]; NULL: no rotation
    const int* positions;
    int table_rows, half;      // half = rot / 2
    int pairs;                 // interleaved pairs instead of halves
};

struct HeadsIn {               // [token][head][dim], strides in elements, dim contiguous
    const void* p;
    long long token, head;
};

struct AppendParams {
    HeadsIn q, k, v, qo;       // qo.p is written
    const int* slots;
    int8_t* kc;
    int8_t* vc;
    float* ks;
    float* vs;
    long long block_stride;    // bytes
    int blocks, kv_heads, shift, dim, tokens, q_heads;
    int q_groups, q_group;     // groups of query heads, heads in one
    int q_ctas, kv_tile;       // CTAs of the queries' part, which come last
    int vec;                   // pointers and strides allow 16-byte accesses
    RopeParams rope;
};

template <bool F32>
__device__ __forceinline__ void load8(const void* base, long long at, bool vec, float (&v)[8]) {
    if constexpr (F32) {
        const float* s = static_cast<const float*>(base) + at;
        if (vec) {
            const float4 a = *reinterpret_cast<const float4*>(s), b = *reinterpret_cast<const float4*>(s + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = s[i];
        }
    } else {
        const __half* s = static_cast<const __half*>(base) + at;
        if (vec) {
            const uint4 a = *reinterpret_cast<const uint4*>(s);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __half2float(s[i]);
        }
    }
}

template <bool F32>
__device__ __forceinline__ void store8(void* base, long long at, bool vec, const float (&v)[8]) {
    if constexpr (F32) {
        float* d = static_cast<float*>(base) + at;
        if (vec) {
            *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = v[i];
        }
    } else {
        __half* d = static_cast<__half*>(base) + at;
        if (vec) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = __float2half_rn(v[i]);
        }
    }
}

// Unit `j` of a head: the element offsets of its two groups of eight (ROTATED units come first).
__device__ __forceinline__ void unit_offsets(const RopeParams& r, int j, int& e0, int& e1, bool& rotated) {
    const int n = r.table ? r.half >> 3 : 0;            // rotated units
    rotated = j < n;
    if (rotated && !r.pairs) { e0 = 8 * j; e1 = r.half + 8 * j; }
    else { e0 = 16 * j; e1 = 16 * j + 8; }              // pairs, and what lies behind the rotated part
}

__device__ __forceinline__ void load_turn(const float2* row, int j, float2 (&cs)[8]) {
    if (row) {
        const float4* s = reinterpret_cast<const float4*>(row + 8 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 t = __ldg(s + i);
            cs[2 * i] = make_float2(t.x, t.y);
            cs[2 * i + 1] = make_float2(t.z, t.w);
        }
    } else {
        const float nan = __int_as_float(0x7fc00000);
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = make_float2(nan, nan);
    }
}

__device__ __forceinline__ void rotate_unit(bool pairs, const float2 (&cs)[8], float (&a)[8], float (&b)[8]) {
    if (pairs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = a[2 * i], y0 = a[2 * i + 1], x1 = b[2 * i], y1 = b[2 * i + 1];
            a[2 * i] = x0 * cs[i].x - y0 * cs[i].y;
            a[2 * i + 1] = y0 * cs[i].x + x0 * cs[i].y;
            b[2 * i] = x1 * cs[i + 4].x - y1 * cs[i + 4].y;
            b[2 * i + 1] = y1 * cs[i + 4].x + x1 * cs[i + 4].y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * cs[i].x - y * cs[i].y;
            b[i] = y * cs[i].x + x * cs[i].y;
        }
    }
}

// The table row of a position; NULL (the rotated part becomes NaN) where it lies outside the table.  That is an error unless the
// row has a slot, and a negative one: the plan gives such to a sequence that it refuses, whose positions may go on behind the table.
__device__ __forceinline__ const float2* rope_row(const RopeParams& r, int pos, const int* slot = nullptr) {
    if (pos < 0 || pos >= r.table_rows) {
        if (!slot || *slot >= 0) report_error(ZTQ_ERR_POSITION);
        return nullptr;
    }
    return r.table + (long long)pos * r.half;
}

template <bool XF32, bool YF32>
__device__ __forceinline__ void rope_heads(const RopeParams& r, const HeadsIn& x, const HeadsIn& y, int t0, int t1, int h0, int h1, int dim, bool vec, const int* slots = nullptr) {
    const int units = dim >> 4, pairs = kTokenTile * units, strides = kRopeThreads / pairs;      // threads of one head: at most the CTA's
    const int at = threadIdx.x % pairs, j = at % units, t = t0 + at / units, first = threadIdx.x / pairs;
    if (first >= strides || t >= t1) return;
    int e0, e1;
    bool rotated;
    unit_offsets(r, j, e0, e1, rotated);
    float2 cs[8];
    if (rotated) load_turn(rope_row(r, r.positions[t], slots ? slots + t : nullptr), j, cs);
    const long long src = t * x.token, dst = t * y.token;
#pragma unroll 4
    for (int h = h0 + first; h < h1; h += strides) {
        float a[8], b[8];
        load8<XF32>(x.p, src + h * x.head + e0, vec, a);
        load8<XF32>(x.p, src + h * x.head + e1, vec, b);
        if (rotated) rotate_unit(r.pairs, cs, a, b);
        store8<YF32>(const_cast<void*>(y.p), dst + h * y.head + e0, vec, a);
        store8<YF32>(const_cast<void*>(y.p), dst + h * y.head + e1, vec, b);
    }
}

// A unit of a new row of keys (rotated) or values.
template <bool XF32>
__device__ __forceinline__ void append_unit(const AppendParams& p, bool key, int t, int pos, int h, int j, float (&a)[8], float (&b)[8], int& e0, int& e1) {
    const HeadsIn& x = key ? p.k : p.v;
    bool rotated = false;
    if (key) unit_offsets(p.rope, j, e0, e1, rotated);
    else { e0 = 16 * j; e1 = 16 * j + 8; }
    const long long src = t * x.token + h * x.head;
    load8<XF32>(x.p, src + e0, p.vec, a);
    load8<XF32>(x.p, src + e1, p.vec, b);
    if (rotated) {
        float2 cs[8];
        load_turn(rope_row(p.rope, pos), j, cs);
        rotate_unit(p.rope.pairs, cs, a, b);
    }
}

// Four codes of v * inv, rounded to nearest even: adding 1.5 2^23 leaves the integer in the low byte.
__device__ __forceinline__ uint32_t pack4(const float* v, float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(fminf(fmaxf(v[i] * inv, -127.f), 127.f) + 12582912.f);
    return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

// The smallest power of two s with amax <= 127 s (not below the smallest normal number); NaN for a non-finite amax.
__device__ __forceinline__ float scale_for(float amax) {
    if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - ((u & 0x7fffffu) <= 0x7e0000u ? 6 : 5);       // 127/64 = 1.984375
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// One run (rows t0 .. t0 + n of a block, from offset `off` of it, at positions pos[0 .. n)) of one head, keys or values, by
// LANES threads: a warp, or the whole CTA with its shared words `red`.
template <bool XF32, int LANES>
__device__ __forceinline__ void append_run(const AppendParams& p, bool key, int h, int t0, const int* pos, int n, int block, int off, int lane, float* red) {
    const int units = p.dim >> 4, size = 1 << p.shift, items = n * units;
    int8_t* codes = (key ? p.kc : p.vc) + block * p.block_stride + (long long)h * size * p.dim;
    float* scale_at = (key ? p.ks : p.vs) + (long long)block * p.kv_heads + h;
    const float had = off > 0 ? *scale_at : 0.f;
    float amax = 0.f;
    bool odd = false;                                  // a NaN: fmaxf would drop it
    int e0, e1;
#pragma unroll 2
    for (int i = lane; i < items; i += LANES) {
        float a[8], b[8];
        const int t = i / units;
        append_unit<XF32>(p, key, t0 + t, pos[t], h, i - t * units, a, b, e0, e1);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            amax = fmaxf(amax, fmaxf(fabsf(a[k]), fabsf(b[k])));
            odd |= a[k] != a[k] || b[k] != b[k];
        }
    }
    if (odd) amax = __int_as_float(0x7f800000);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if constexpr (LANES > 32) {
        __syncthreads();                               // the previous run's readers are done with red; everyone has read `had`
        if ((lane & 31) == 0) red[lane >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < LANES / 32; ++w) amax = fmaxf(amax, red[w]);
    }
    const float need = scale_for(amax);
    float scale = need;
    if (off > 0 && !(need != need)) scale = had != had ? had : fmaxf(had, need);
    const bool dead = scale != scale;
    if (off > 0 && !dead && scale != had) {            // the block's scale grows: its rows are rounded to the new step
        const float ratio = had / scale;
        for (int i = lane; i < off * units; i += LANES) {
            uint4 w = *reinterpret_cast<const uint4*>(codes + 16 * i);
            uint32_t* q = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) v[m] = (float)(int8_t)(q[k] >> (8 * m));
                q[k] = pack4(v, ratio);
            }
            *reinterpret_cast<uint4*>(codes + 16 * i) = w;
        }
    }
    // A power of two's reciprocal is exact; a scale from elsewhere that stays (the append writes powers of two) costs one
    // more rounding of 2^-24.  Dead blocks get code 0.
    const float inv = 1.f / scale;
    for (int i = lane; i < items; i += LANES) {
        float a[8], b[8];
        const int t = i / units;
        append_unit<XF32>(p, key, t0 + t, pos[t], h, i - t * units, a, b, e0, e1);
        int8_t* row = codes + (long long)(off + t) * p.dim;
        *reinterpret_cast<uint2*>(row + e0) = dead ? make_uint2(0, 0) : make_uint2(pack4(a, inv), pack4(a + 4, inv));
        *reinterpret_cast<uint2*>(row + e1) = dead ? make_uint2(0, 0) : make_uint2(pack4(b, inv), pack4(b + 4, inv));
    }
    if (lane == 0) *scale_at = scale;
}

template <bool XF32, bool YF32>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_append_kernel(const AppendParams p) {
    constexpr int kSeen = kMaxKvTile + 128;            // rows that a run of the tile may reach
    __shared__ int s_slot[kSeen + 1], s_pos[kSeen], s_run[kMaxKvTile], s_count;
    __shared__ float red[kRopeThreads / 32];
    grid_dep_launch();
    grid_dep_wait();
    const int kv_parts = 2 * p.kv_heads, kv_ctas = (int)gridDim.x - p.q_ctas;
    if ((int)blockIdx.x >= kv_ctas) {
        const int at = blockIdx.x - kv_ctas, t0 = at / p.q_groups * kTokenTile, h0 = at % p.q_groups * p.q_group;
        rope_heads<XF32, YF32>(p.rope, p.q, p.qo, t0, min(t0 + kTokenTile, p.tokens), h0, min(h0 + p.q_group, p.q_heads), p.dim, p.vec, p.slots);
        return;
    }
    const int tile = blockIdx.x / kv_parts, which = blockIdx.x % kv_parts, t0 = tile * p.kv_tile;
    const int h = which >> 1, size = 1 << p.shift, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool key = !(which & 1);
    const long long limit = (long long)p.blocks << p.shift;
    // slots and positions of all rows that matter here, in one go; s_slot[0] is the row in front of the tile
    if (tid < p.kv_tile + size && tid < kSeen) {
        const int t = t0 + tid;
        s_slot[tid + 1] = t < p.tokens ? p.slots[t] : -1;
        s_pos[tid] = key && p.rope.table && t < p.tokens ? p.rope.positions[t] : 0;
    }
    if (tid == kRopeThreads - 1) { s_slot[0] = t0 > 0 ? p.slots[t0 - 1] : -1; s_count = 0; }
    __syncthreads();
    if (tid < p.kv_tile) {                             // rows of this tile that begin a run
        const int s = s_slot[tid + 1], before = s_slot[tid];
        bool begins = s >= 0 && s < limit;
        if (s >= limit) report_error(ZTQ_ERR_SLOT);
        if (begins && before >= 0 && (before >> p.shift) == (s >> p.shift)) {
            begins = false;
            if (s != before + 1) report_error(ZTQ_ERR_SLOT);               // and the run in front ends there
        }
        if (begins) s_run[atomicAdd(&s_count, 1)] = tid;
    }
    __syncthreads();
    const int runs = s_count;
    const bool shared = runs < kRopeThreads / 32;
    for (int i = shared ? 0 : warp; i < runs; i += shared ? 1 : kRopeThreads / 32) {
        const int at = s_run[i], s = s_slot[at + 1], off = s & (size - 1);
        int n = 1;                                     // rows of the run: 32 candidates at a time
        while (off + n < size) {
            const int u = n + lane;
            const bool goes_on = off + u < size && s_slot[at + 1 + u] == s + u;
            const unsigned miss = ~__ballot_sync(0xffffffffu, goes_on);
            n += miss ? __ffs(miss) - 1 : 32;
            if (miss) break;
        }
        if (shared) append_run<XF32, kRopeThreads>(p, key, h, t0 + at, s_pos + at, n, s >> p.shift, off, tid, red);
        else append_run<XF32, 32>(p, key, h, t0 + at, s_pos + at, n, s >> p.shift, off, lane, red);
    }
}

template <bool XF32, bool YF32>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams r, const HeadsIn x, const HeadsIn y, int tokens, int heads, int group, int dim, int vec) {
    grid_dep_launch();
    grid_dep_wait();
    const int t0 = blockIdx.x * kTokenTile, h0 = blockIdx.y * group;
    rope_heads<XF32, YF32>(r, x, y, t0, min(t0 + kTokenTile, tokens), h0, min(h0 + group, heads), dim, vec);
}

// Table of {cos, sin} of positions first .. first + rows: angles in 64 bits, one rounding to fp32.
constexpr int kRopeMaxHalf = 128;
struct RopeFreq {
    double f[kRopeMaxHalf];
    double magnitude;
};
__global__ void rope_table_kernel(float2* table, int first, long long rows, int half, const __grid_constant__ RopeFreq fr) {
    grid_dep_launch();
    grid_dep_wait();
    const long long n = rows * half;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        double s, c;
        sincos((double)(first + i / half) * fr.f[i % half], &s, &c);
        table[i] = make_float2((float)(c * fr.magnitude), (float)(s * fr.magnitude));
    }
}

// Cache rows -> fp16 or fp32 [rows][kv_heads][dim]; a slot outside the cache leaves its row as it was.
template <bool YF32>
__global__ void __launch_bounds__(kRopeThreads) kv_read_kernel(const AppendParams p, void* k_out, void* v_out) {
    grid_dep_launch();
    grid_dep_wait();
    const int units = p.dim >> 4, size = 1 << p.shift;
    const int per = p.kv_heads * units;
    const long long n = (long long)p.tokens * per, limit = (long long)p.blocks << p.shift;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int t = n < 0x7fffffff ? (int)((unsigned)i / (unsigned)per) : (int)(i / per);     // a 64-bit division costs more than the copy
        const int rest = (int)(i - (long long)t * per), h = rest / units, j = rest % units;
        const int s = p.slots[t];
        if (s < 0 || s >= limit) continue;
        const int block = s >> p.shift;
        const long long at = block * p.block_stride + ((long long)h * size + (s & (size - 1))) * p.dim + 16 * j;
        const long long to = (t * (long long)p.kv_heads + h) * p.dim + 16 * j;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            void* out = w ? v_out : k_out;
            if (!out) continue;
            const uint4 c = *reinterpret_cast<const uint4*>((w ? p.vc : p.kc) + at);
            const float scale = (w ? p.vs : p.ks)[(long long)block * p.kv_heads + h];
            const uint32_t q[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float v[8];
#pragma unroll
                for (int m = 0; m < 8; ++m) v[m] = (float)(int8_t)(q[2 * g + (m >> 2)] >> (8 * (m & 3))) * scale;
                store8<YF32>(out, to + 8 * g, true, v);
            }
        }
    }
}

}  // namespace ztq
