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
// Work: units of 16 elements of one head.  A CTA holds a tile of kTokenTile rows; blockIdx.y is a group of query heads
// or a key/value head.  The rows of one block stand together (a run); the CTA whose tile holds a run's first row does
// the whole run, so a block has one writer and needs no atomics.  With few runs in the tile (a prompt) the CTA's warps
// share each run, with many (decoding) every warp takes runs of its own.
#pragma once

#include "ztq_common.cuh"

namespace ztq {

constexpr int kRopeThreads = 256;
constexpr int kTokenTile = 16;

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
    int x_f32, y_f32, vec;     // vec: pointers and strides allow 16-byte accesses
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

__device__ __forceinline__ void rotate_unit(const RopeParams& r, const float2* row, int j, float (&a)[8], float (&b)[8]) {
    float2 cs[8];
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
    if (r.pairs) {
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

// The table row of a token; NULL (the rotated part becomes NaN) where its position lies outside the table.
__device__ __forceinline__ const float2* rope_row(const RopeParams& r, int token) {
    const int pos = r.positions[token];
    if (pos < 0 || pos >= r.table_rows) {
        report_error(ZTQ_ERR_POSITION);
        return nullptr;
    }
    return r.table + (long long)pos * r.half;
}

template <bool XF32, bool YF32>
__device__ __forceinline__ void rope_heads(const RopeParams& r, const HeadsIn& x, const HeadsIn& y, int t0, int t1, int h0, int h1, int dim, bool vec) {
    const int units = dim >> 4, heads = h1 - h0;
    for (int i = threadIdx.x; i < (t1 - t0) * heads * units; i += blockDim.x) {
        const int j = i % units, h = h0 + i / units % heads, t = t0 + i / (units * heads);
        int e0, e1;
        bool rotated;
        unit_offsets(r, j, e0, e1, rotated);
        const long long src = t * x.token + h * x.head, dst = t * y.token + h * y.head;
        float a[8], b[8];
        load8<XF32>(x.p, src + e0, vec, a);
        load8<XF32>(x.p, src + e1, vec, b);
        if (rotated) rotate_unit(r, rope_row(r, t), j, a, b);
        store8<YF32>(const_cast<void*>(y.p), dst + e0, vec, a);
        store8<YF32>(const_cast<void*>(y.p), dst + e1, vec, b);
    }
}

// A unit of a new row of keys (rotated) or values.
template <bool XF32>
__device__ __forceinline__ void append_unit(const AppendParams& p, bool key, int t, int h, int j, float (&a)[8], float (&b)[8], int& e0, int& e1) {
    const HeadsIn& x = key ? p.k : p.v;
    bool rotated = false;
    if (key) unit_offsets(p.rope, j, e0, e1, rotated);
    else { e0 = 16 * j; e1 = 16 * j + 8; }
    const long long src = t * x.token + h * x.head;
    load8<XF32>(x.p, src + e0, p.vec, a);
    load8<XF32>(x.p, src + e1, p.vec, b);
    if (rotated) rotate_unit(p.rope, rope_row(p.rope, t), j, a, b);
}

__device__ __forceinline__ uint32_t pack4(const float* v, float inv, bool dead) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = dead ? 0 : __float2int_rn(fminf(fmaxf(v[i] * inv, -127.f), 127.f));
        w |= (uint32_t)(c & 255) << (8 * i);
    }
    return w;
}

// The smallest power of two s with amax <= 127 s (not below the smallest normal number); NaN for a non-finite amax.
__device__ __forceinline__ float scale_for(float amax) {
    if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - ((u & 0x7fffffu) <= 0x7e0000u ? 6 : 5);       // 127/64 = 1.984375
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// One run (rows t0 .. t0 + n of a block, from offset `off` of it) of one head, keys or values, by a group of `lanes`
// threads (a warp, or the whole CTA with its shared word `red`).
template <bool XF32>
__device__ __forceinline__ void append_run(const AppendParams& p, bool key, int h, int t0, int n, int block, int off, int lane, int lanes, float* red) {
    const int units = p.dim >> 4, size = 1 << p.shift;
    int8_t* codes = (key ? p.kc : p.vc) + block * p.block_stride + (long long)h * size * p.dim;
    float* scale_at = (key ? p.ks : p.vs) + (long long)block * p.kv_heads + h;
    const float had = *scale_at;
    float amax = 0.f;
    bool odd = false;                                  // a NaN: fmaxf would drop it
    int e0, e1;
    for (int i = lane; i < n * units; i += lanes) {
        float a[8], b[8];
        append_unit<XF32>(p, key, t0 + i / units, h, i % units, a, b, e0, e1);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            amax = fmaxf(amax, fmaxf(fabsf(a[k]), fabsf(b[k])));
            odd |= a[k] != a[k] || b[k] != b[k];
        }
    }
    if (odd) amax = __int_as_float(0x7f800000);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lanes > 32) {
        __syncthreads();                               // the previous run's readers are done with red, and everyone has read `had`
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
        __syncthreads();
        for (int w = 0; w < (lanes >> 5); ++w) amax = fmaxf(amax, red[w]);
    }
    const float need = scale_for(amax);
    float scale = need;
    if (off > 0 && !(need != need)) scale = had != had ? had : fmaxf(had, need);
    const bool dead = scale != scale;
    if (off > 0 && !dead && scale != had) {            // the block's scale grows: its rows are rounded to the new step
        const float ratio = had / scale;
        for (int i = lane; i < off * units; i += lanes) {
            uint4 w = *reinterpret_cast<const uint4*>(codes + 16 * i);
            uint32_t* q = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) v[m] = (float)(int8_t)(q[k] >> (8 * m));
                q[k] = pack4(v, ratio, false);
            }
            *reinterpret_cast<uint4*>(codes + 16 * i) = w;
        }
    }
    // 1 / scale of a power of two is exact, but below 2^-126 for the largest scales: division by it is not
    const float inv = 1.f / scale;
    for (int i = lane; i < n * units; i += lanes) {
        float a[8], b[8];
        const int t = i / units;
        append_unit<XF32>(p, key, t0 + t, h, i % units, a, b, e0, e1);
        int8_t* row = codes + (long long)(off + t) * p.dim;
        *reinterpret_cast<uint2*>(row + e0) = make_uint2(pack4(a, inv, dead), pack4(a + 4, inv, dead));
        *reinterpret_cast<uint2*>(row + e1) = make_uint2(pack4(b, inv, dead), pack4(b + 4, inv, dead));
    }
    if (lane == 0) *scale_at = scale;
}

template <bool XF32, bool YF32>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const AppendParams p) {
    __shared__ int s_run[kTokenTile], s_count;
    __shared__ float red[kRopeThreads / 32];
    grid_dep_launch();
    grid_dep_wait();
    const int t0 = blockIdx.x * kTokenTile, t1 = min(t0 + kTokenTile, p.tokens);
    if ((int)blockIdx.y < p.q_groups) {
        const int h0 = blockIdx.y * p.q_group;
        rope_heads<XF32, YF32>(p.rope, p.q, p.qo, t0, t1, h0, min(h0 + p.q_group, p.q_heads), p.dim, p.vec);
        return;
    }
    const int h = blockIdx.y - p.q_groups, size = 1 << p.shift;
    const long long limit = (long long)p.blocks << p.shift;
    if (threadIdx.x < 32) {
        // rows of this tile that begin a run
        const int t = t0 + threadIdx.x;
        bool begins = false;
        if (threadIdx.x < kTokenTile && t < t1) {
            const int s = p.slots[t], before = t > 0 ? p.slots[t - 1] : -1;
            begins = s >= 0 && s < limit;
            if (s >= limit) report_error(ZTQ_ERR_SLOT);
            if (begins && before >= 0 && (before >> p.shift) == (s >> p.shift)) {
                begins = false;
                if (s != before + 1) report_error(ZTQ_ERR_SLOT);           // and append_run's count stops in front of it
            }
        }
        const unsigned found = __ballot_sync(0xffffffffu, begins);
        if (begins) s_run[__popc(found & ((1u << threadIdx.x) - 1))] = t;
        if (threadIdx.x == 0) s_count = __popc(found);
    }
    __syncthreads();
    const int runs = s_count, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool shared = 2 * runs < kRopeThreads / 32;
    for (int i = shared ? 0 : warp; i < 2 * runs; i += shared ? 1 : kRopeThreads / 32) {
        const int t = s_run[i >> 1], s = p.slots[t], off = s & (size - 1);
        int n = 1;                                     // rows of the run: 32 candidates at a time
        while (off + n < size) {
            const int u = t + n + lane;
            const bool goes_on = u < p.tokens && off + n + lane < size && p.slots[u] == s + n + lane;
            const unsigned miss = ~__ballot_sync(0xffffffffu, goes_on);
            n += miss ? __ffs(miss) - 1 : 32;
            if (miss) break;
        }
        append_run<XF32>(p, !(i & 1), h, t, n, s >> p.shift, off, shared ? threadIdx.x : lane, shared ? kRopeThreads : 32, red);
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
    const long long per = (long long)p.kv_heads * units, n = p.tokens * per, limit = (long long)p.blocks << p.shift;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int t = (int)(i / per), h = (int)(i % per) / units, j = (int)(i % units);
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
