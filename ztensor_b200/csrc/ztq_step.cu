// ztq_step.cu -- extern "C" launchers of the decode-step operators around the projections (see include/ztq.h):
// the step plan, rotary positions and the append to the 8-bit cache, sampling.
#include "../../include/ztq.h"

#include "kv_plan.cuh"
#include "launch.cuh"
#include "rope_append.cuh"
#include "sample.cuh"

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace ztq {

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool ready() { return device_info().major >= 10; }

// log2 of a block size the cache allows, or -1
static int block_shift(int block_size) {
    for (int s = 4; s <= 7; ++s)
        if (block_size == 1 << s) return s;
    return -1;
}

static bool cache_ok(const ZtqKvCache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || c->blocks <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535) return false;
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16) return false;
    const int shift = block_shift(c->block_size);
    if (shift < 0 || (long long)c->blocks << shift > 0x7fffffffll) return false;
    if (c->block_stride < (long long)c->kv_heads * c->block_size * c->head_dim || c->block_stride % 16) return false;
    return aligned16(c->k) && aligned16(c->v);
}

// Rotary arguments -> parameters; false where they do not fit heads of `dim`.
static bool rope_params(const void* table, int table_rows, int rot_dim, const int* positions, int tokens, int dim, int flags, RopeParams& r) {
    r = RopeParams{};
    if (!table) return true;
    if (!aligned16(table) || table_rows <= 0 || rot_dim < 16 || rot_dim % 16 || rot_dim > dim || (tokens != 0 && !positions)) return false;
    r.table = static_cast<const float2*>(table);
    r.positions = positions;
    r.table_rows = table_rows;
    r.half = rot_dim / 2;
    r.pairs = (flags & ZTQ_ROPE_PAIRS) ? 1 : 0;
    return true;
}

static bool wide(const HeadsIn& x, bool f32) {
    const int n = f32 ? 4 : 8;
    return aligned16(x.p) && x.token % n == 0 && x.head % n == 0;
}

// Query heads a CTA takes: all of them once the row tiles fill the device, else as few as its threads hold at a time
static int head_group(int heads, int tiles, int dim, int sms) {
    const int least = std::max(1, kRopeThreads / (kTokenTile * (dim / 16)));
    int group = heads;
    while (group > least && (long long)tiles * ceil_div(heads, group) < 4ll * sms) group = (group + 1) / 2;
    return group;
}

}  // namespace ztq

using namespace ztq;

extern "C" {

int ztq_take_error_step() { return take_error(); }

cudaError_t ztq_kv_plan(const int* ctx_len, const int* new_len, int* block_table, int* ring, const int* ring_state, int* ring_state_out,
                        int* next_len, int* kv_len, int* query_start, int* positions, int* slots, int* status, int sequences, int table_width,
                        int block_size, int pool_blocks, int max_tokens, int flags, cudaStream_t stream) {
    const int shift = block_shift(block_size);
    if (!ctx_len || !new_len || !block_table || !ring || !ring_state || !ring_state_out || !next_len || !kv_len || !query_start || !positions || !slots || !status)
        return cudaErrorInvalidValue;
    if (sequences <= 0 || sequences > kPlanMaxSeqs || table_width <= 0 || shift < 0 || pool_blocks <= 0 || max_tokens <= 0) return cudaErrorInvalidValue;
    if ((long long)table_width << shift > 0x7fffffffll || (long long)pool_blocks << shift > 0x7fffffffll) return cudaErrorInvalidValue;
    if (flags & ~ZTQ_NO_PDL) return cudaErrorInvalidValue;
    if (!ready()) return cudaErrorNoKernelImageForDevice;
    const PlanParams p{ctx_len, new_len, block_table, ring, ring_state, ring_state_out, next_len, kv_len, query_start, positions, slots, status,
                       sequences, table_width, shift, pool_blocks, max_tokens};
    static std::atomic<unsigned> done{0};
    if (cudaError_t e = allow_smem(kv_plan_kernel, done, kPlanMaxSeqs * 28 + 64)) return e;
    // one CTA per 1024 rows or 128 sequences, as far as a cluster goes
    int ctas = max(ceil_div(max_tokens, kPlanThreads), ceil_div(sequences, 128)), n = 1;
    while (n < ctas && n < 8) n *= 2;
    const size_t smem = (size_t)sequences * sizeof(PlanSeq) + (sequences + 1) * 4;
    cudaError_t e = launch_cluster(kv_plan_kernel, dim3(n), n, dim3(kPlanThreads), smem, stream, !(flags & ZTQ_NO_PDL), p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t ztq_rope_table(void* table, int first, int rows, const ZtqRopeSpec* s, int flags, cudaStream_t stream) {
    if (!table || !aligned16(table) || !s || rows <= 0 || first < 0 || rows > 0x7fffffff - first || (flags & ~ZTQ_NO_PDL)) return cudaErrorInvalidValue;
    if (s->rot_dim < 16 || s->rot_dim % 16 || s->rot_dim > 2 * kRopeMaxHalf || !(s->base > 0) || !std::isfinite(s->base)) return cudaErrorInvalidValue;
    if (s->scaling != ZTQ_ROPE_UNSCALED && (!(s->factor > 0) || !std::isfinite(s->factor))) return cudaErrorInvalidValue;
    RopeFreq f;
    f.magnitude = s->magnitude == 0 ? 1.0 : s->magnitude;
    if (!std::isfinite(f.magnitude)) return cudaErrorInvalidValue;
    const double pi = 3.14159265358979323846;
    for (int i = 0; i < s->rot_dim / 2; ++i) {
        double w = std::pow(s->base, -2.0 * i / s->rot_dim);
        if (s->scaling == ZTQ_ROPE_LINEAR) w /= s->factor;
        if (s->scaling == ZTQ_ROPE_BY_TURNS) {
            // turns the frequency makes over the original context: many -> kept, few -> stretched, a ramp between
            if (!(s->turns_high > s->turns_low) || !(s->original_positions > 0)) return cudaErrorInvalidValue;
            const double turns = s->original_positions * w / (2 * pi);
            double keep = (turns - s->turns_low) / (s->turns_high - s->turns_low);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            w = w * keep + w / s->factor * (1 - keep);
        } else if (s->scaling == ZTQ_ROPE_BY_DIM) {
            // the same ramp drawn over the dimension ("NTK-by-parts", Peng et al., YaRN, 2023, with its 0.001 against a ramp of no width): linear in i between the dimensions that make turns_high and turns_low turns
            if (!(s->turns_high > s->turns_low) || !(s->turns_low > 0) || !(s->original_positions > 0) || !(s->base > 1)) return cudaErrorInvalidValue;
            auto dim_of = [&](double turns) { return s->rot_dim * std::log(s->original_positions / (turns * 2 * pi)) / (2 * std::log(s->base)); };
            double a = std::floor(dim_of(s->turns_high)), b = std::ceil(dim_of(s->turns_low));
            a = a < 0 ? 0 : a;
            b = b > s->rot_dim - 1 ? s->rot_dim - 1 : b;
            if (b <= a) b = a + 0.001;
            double stretch = (i - a) / (b - a);
            stretch = stretch < 0 ? 0 : stretch > 1 ? 1 : stretch;
            w = w * (1 - stretch) + w / s->factor * stretch;
        } else if (s->scaling != ZTQ_ROPE_UNSCALED && s->scaling != ZTQ_ROPE_LINEAR) return cudaErrorInvalidValue;
        f.f[i] = w;
    }
    if (!ready()) return cudaErrorNoKernelImageForDevice;
    const long long n = (long long)rows * (s->rot_dim / 2);
    const int grid = (int)(n / 256 + 1 < 16 * 148 ? n / 256 + 1 : 16 * 148);
    cudaError_t e = launch(rope_table_kernel, dim3(grid), dim3(256), 0, stream, !(flags & ZTQ_NO_PDL), static_cast<float2*>(table), first, (long long)rows, s->rot_dim / 2, f);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t ztq_rope(const void* x, void* y, int tokens, int heads, int head_dim, long long x_token, long long x_head, long long y_token,
                     long long y_head, const void* table, int table_rows, int rot_dim, const int* positions, int flags, cudaStream_t stream) {
    if ((tokens != 0 && (!x || !y)) || tokens < 0 || heads <= 0 || head_dim < 16 || head_dim > 256 || head_dim % 16 || !table) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_NO_PDL | ZTQ_ROPE_PAIRS)) return cudaErrorInvalidValue;
    RopeParams r;
    if (!rope_params(table, table_rows, rot_dim, positions, tokens, head_dim, flags, r)) return cudaErrorInvalidValue;
    const bool xf = flags & ZTQ_X_F32, yf = flags & ZTQ_Y_F32;
    if (x && x == y && (xf != yf || x_token != y_token || x_head != y_head)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    if (tokens == 0) return cudaSuccess;
    const HeadsIn in{x, x_token, x_head}, out{y, y_token, y_head};
    const int vec = wide(in, xf) && wide(out, yf);
    const int tiles = ceil_div(tokens, kTokenTile), group = max(head_group(heads, tiles, head_dim, dev.sms), ceil_div(heads, 65535));
    const dim3 grid(tiles, ceil_div(heads, group));
    auto kern = xf ? (yf ? rope_kernel<true, true> : rope_kernel<true, false>) : (yf ? rope_kernel<false, true> : rope_kernel<false, false>);
    cudaError_t e = launch(kern, grid, dim3(kRopeThreads), 0, stream, !(flags & ZTQ_NO_PDL), r, in, out, tokens, heads, group, head_dim, vec);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t ztq_rope_append_q8(const void* q, const void* k, const void* v, void* q_out, long long q_token, long long q_head, long long k_token,
                               long long k_head, long long v_token, long long v_head, long long qo_token, long long qo_head, int tokens, int q_heads,
                               const void* table, int table_rows, int rot_dim, const int* positions, const int* slots, const ZtqKvCache* cache,
                               int flags, cudaStream_t stream) {
    if ((tokens != 0 && (!k || !v || !slots || (q_heads > 0 && (!q || !q_out)))) || tokens < 0 || q_heads < 0 || !cache_ok(cache)) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_NO_PDL | ZTQ_ROPE_PAIRS)) return cudaErrorInvalidValue;
    AppendParams p = {};
    if (!rope_params(table, table_rows, rot_dim, positions, tokens, cache->head_dim, flags, p.rope)) return cudaErrorInvalidValue;
    const bool xf = flags & ZTQ_X_F32, yf = flags & ZTQ_Y_F32;
    if (q_heads > 0 && q && q == q_out && (xf != yf || q_token != qo_token || q_head != qo_head)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    if (tokens == 0) return cudaSuccess;
    p.q = HeadsIn{q, q_token, q_head};
    p.k = HeadsIn{k, k_token, k_head};
    p.v = HeadsIn{v, v_token, v_head};
    p.qo = HeadsIn{q_out, qo_token, qo_head};
    p.slots = slots;
    p.kc = static_cast<int8_t*>(cache->k);
    p.vc = static_cast<int8_t*>(cache->v);
    p.ks = cache->k_scale;
    p.vs = cache->v_scale;
    p.block_stride = cache->block_stride;
    p.blocks = cache->blocks;
    p.kv_heads = cache->kv_heads;
    p.shift = block_shift(cache->block_size);
    p.dim = cache->head_dim;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.vec = wide(p.k, xf) && wide(p.v, xf) && (q_heads == 0 || (wide(p.q, xf) && wide(p.qo, yf)));
    const int tiles = ceil_div(tokens, kTokenTile);
    p.q_group = q_heads ? head_group(q_heads, tiles, p.dim, dev.sms) : 1;
    p.q_groups = q_heads ? ceil_div(q_heads, p.q_group) : 0;
    // tiles of 16 / 64 rows, with the read-back: a prompt of 256 11.2 / 11.8 us, 1024 16.2 / 15.1, 8192 79 / 71; 256 decoding rows 22 / 36,
    // 1024 67 / 77, 2048 128 / 127
    p.kv_tile = tokens >= 16 * kMaxKvTile ? kMaxKvTile : kTokenTile;
    const long long q_ctas = (long long)tiles * p.q_groups, ctas = q_ctas + (long long)ceil_div(tokens, p.kv_tile) * 2 * p.kv_heads;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    p.q_ctas = (int)q_ctas;
    const dim3 grid((unsigned)ctas);
    auto kern = xf ? (yf ? rope_append_kernel<true, true> : rope_append_kernel<true, false>) : (yf ? rope_append_kernel<false, true> : rope_append_kernel<false, false>);
    cudaError_t e = launch(kern, grid, dim3(kRopeThreads), 0, stream, !(flags & ZTQ_NO_PDL), p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t ztq_kv_read_q8(const ZtqKvCache* cache, const int* slots, int tokens, void* k_out, void* v_out, int flags, cudaStream_t stream) {
    if (!cache_ok(cache) || (tokens != 0 && (!slots || (!k_out && !v_out))) || tokens < 0 || !aligned16(k_out) || !aligned16(v_out)) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_Y_F32 | ZTQ_NO_PDL)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    if (tokens == 0) return cudaSuccess;
    AppendParams p = {};
    p.slots = slots;
    p.kc = static_cast<int8_t*>(cache->k);
    p.vc = static_cast<int8_t*>(cache->v);
    p.ks = cache->k_scale;
    p.vs = cache->v_scale;
    p.block_stride = cache->block_stride;
    p.blocks = cache->blocks;
    p.kv_heads = cache->kv_heads;
    p.shift = block_shift(cache->block_size);
    p.dim = cache->head_dim;
    p.tokens = tokens;
    const long long n = (long long)tokens * p.kv_heads * (p.dim / 16), most = 8ll * dev.sms;
    const int grid = (int)((n + kRopeThreads - 1) / kRopeThreads < most ? (n + kRopeThreads - 1) / kRopeThreads : most);
    auto kern = (flags & ZTQ_Y_F32) ? kv_read_kernel<true> : kv_read_kernel<false>;
    cudaError_t e = launch(kern, dim3(grid), dim3(kRopeThreads), 0, stream, !(flags & ZTQ_NO_PDL), p, k_out, v_out);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t ztq_sample(const void* logits, long long row_stride, int rows, int vocab, const float* temperature, const int* top_k,
                       const float* top_p, const float* min_p, const float* uniform, int* token, float* logprob, int flags, cudaStream_t stream) {
    if ((rows != 0 && (!logits || !uniform || !token)) || rows < 0 || vocab <= 0 || vocab > ZTQ_SAMPLE_MAX_VOCAB || (rows > 1 && row_stride < vocab)) return cudaErrorInvalidValue;
    if (rows > 0x7fffffff / kSampleMaxCluster) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_X_F32 | ZTQ_NO_PDL)) return cudaErrorInvalidValue;
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    if (rows == 0) return cudaSuccess;
    const bool f32 = flags & ZTQ_X_F32;
    // CTAs of a row: as many as keep a slice in 64 KB (two CTAs per SM), then twice as many as long as all of them still
    // run at once and a slice is worth a CTA
    auto slice_of = [&](int ranks) { return ceil_div(ceil_div(vocab, ranks), kSampleSeg) * kSampleSeg; };
    int ranks = 1;
    while (ranks < kSampleMaxCluster && slice_of(ranks) * (f32 ? 4 : 2) > 64 * 1024) ranks *= 2;
    while (ranks < kSampleMaxCluster && (long long)rows * ranks <= dev.sms && slice_of(ranks) > 2048) ranks *= 2;
    SampleParams p{logits, row_stride, temperature, top_k, top_p, min_p, uniform, token, logprob, rows, vocab, slice_of(ranks), ranks,
                   aligned16(logits) && row_stride % (f32 ? 4 : 8) == 0};
    const size_t smem = ((sizeof(SampleShared) + 15) & ~15) + (size_t)p.slice * (f32 ? 4 : 2);
    auto kern = f32 ? sample_kernel<true> : sample_kernel<false>;
    static std::atomic<unsigned> done[2];
    if (cudaError_t e = allow_smem(kern, done[f32])) return e;
    cudaError_t e = launch_cluster(kern, dim3(rows * ranks), ranks, dim3(kSampleThreads), smem, stream, !(flags & ZTQ_NO_PDL), p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // extern "C"
