// ztq_attn.cu -- extern "C" launchers of the attention over the paged 8-bit cache (see include/ztq.h).
#include "../../include/ztq.h"

#include "attn_q8.cuh"
#include "attn_tc.cuh"
#include "launch.cuh"

#include <algorithm>
#include <cstdint>
#include <cstring>

namespace ztq {

// Row tiles of eight that a CTA of attn_rows_kernel takes at a time: two where its registers hold them.
static int attn_nt(int head_dim, long long rows, bool split) { return rows <= 8 || head_dim > 128 || (split && head_dim > 64) ? 1 : 2; }

// One layer's keys or values as (dim, head and token, block), copied a block of one head at a time.
static bool cache_map(CUtensorMap* map, const void* base, const AttnParams& p, int dim) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)p.kv_heads << p.shift, (cuuint64_t)p.blocks}, strides[2] = {(cuuint64_t)dim, (cuuint64_t)p.block_stride};
    const cuuint32_t box[3] = {(cuuint32_t)std::min(dim, 128), 1u << p.shift, 1}, ones[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
               dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT, bool SPLIT>
static cudaError_t launch_rows(const AttnParams& p, int sms, cudaStream_t stream, bool pdl) {
    CUtensorMap k_map, v_map;
    if (!cache_map(&k_map, p.kc, p, D) || !cache_map(&v_map, p.vc, p, D)) return cudaErrorInvalidValue;
    static std::atomic<unsigned> done{0};
    auto kern = attn_rows_kernel<D, NT, SPLIT>;
    using Ring = AttnRing<D, NT, SPLIT>;
    const int smem = Ring::bytes(p.seqs);
    if (cudaError_t e = allow_smem(kern, done, Ring::bytes(kAttnMaxSeqs))) return e;
    cudaError_t e = launch(kern, dim3(sms), dim3(Ring::kThreads), smem, stream, pdl, k_map, v_map, p);
    if (e != cudaSuccess || sms < 2) return e;
    // many parts per row: a CTA per row; else a warp per row (sequences of 8000 tokens, 64 / 8 heads of 128, warp / CTA: one 19.8 / 17.8 us,
    // two 20.3 / 20.4, four 22.7 / 24.1, eight 27.4 / 29.5)
    const bool few = (long long)p.seqs * p.kv_heads <= 32;
    e = launch(attn_join_kernel<D, NT>, dim3(sms - 1, few ? 8 * NT : NT), dim3(kJoinThreads), p.seqs * 8, stream, pdl, p, sms);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <int D>
static cudaError_t launch_dim(const AttnParams& p, int nt, bool split, int sms, cudaStream_t stream, bool pdl) {
    if constexpr (D == 64) {
        if (nt == 2 && split) return launch_rows<D, 2, true>(p, sms, stream, pdl);
    }
    if constexpr (D <= 128) {
        if (nt == 2) return launch_rows<D, 2, false>(p, sms, stream, pdl);
    }
    return split ? launch_rows<D, 1, true>(p, sms, stream, pdl) : launch_rows<D, 1, false>(p, sms, stream, pdl);
}

// Prompts: sequences with more than kTcMinRows rows per kv head go to the tensor-core kernel (heads of 64 and 128).
// Over 3000 tokens with 64 / 8 heads of 128 in fp16, attn_rows_kernel / attn_tc_kernel: 64 sequences of 64 rows per kv head 272 / 384 us, of 96
// 350 / 381, of 128 522 / 383; four sequences of 64 rows 33 / 72, of 128 47 / 52, of 192 71 / 65.  With 32 / 8 heads of 64 the rows
// kernel stays ahead longer (64 sequences of 96 rows 249 / 358).
// With few sequences all of them do: a launch of its own for those with few rows would cost more than their 256-row items
// (three sequences of 91, 26 and 91 tokens: 58 us with both kernels and their joins, 33 with one).
constexpr int kTcMinRows = 64;

struct TcPlan {
    long long items = 0;          // CTAs of one split; 0: the kernel is not used
    int splits = 1;
    bool all = false;             // takes every sequence
    size_t bytes = 0;             // of its workspace
};
static TcPlan tc_plan(int tokens, int sequences, long long most_rows, int group, int kv_heads, int head_dim, bool split, int sms) {
    TcPlan t;
    if (most_rows <= kTcMinRows || head_dim > 128) return t;
    t.all = sequences == 1 || (long long)sequences * kv_heads <= sms;
    // items: full ones, and one begun by each sequence that is taken
    const long long rows = (long long)tokens * group, full = rows / tca_rows(split);
    const long long begun = t.all ? sequences : std::min<long long>(sequences, rows / (kTcMinRows + 1) + 1);
    t.items = (full + begun) * kv_heads;
    // few items: cut their keys so that every SM has a CTA.  Half the begun ones are taken to be there: counting on fewer
    // would make the workspace (items x splits) grow with the square of the sequences
    const long long few = std::max(full, (begun + 1) / 2) * kv_heads;
    if (few < sms) t.splits = (int)std::min<long long>(sms / few, 32);
    if (t.splits > 1) t.bytes = (size_t)t.items * t.splits * tca_rows(split) * (head_dim + 2) * sizeof(float);
    return t;
}

template <int D, bool SPLIT>
static cudaError_t launch_tc(const AttnParams& p, const TcPlan& plan, cudaStream_t stream, bool pdl) {
    TcaParams tp;
    tp.a = p;
    // a split is worth eight steps: the join takes as long as two
    tp.splits = (int)std::max<long long>(1, std::min<long long>(plan.splits, ((long long)p.width << p.shift) / (8 * kTcaKeys)));
    tp.rows = tca_rows(SPLIT);
    tp.parts = p.parts;
    static std::atomic<unsigned> done{0};
    auto kern = attn_tc_kernel<D, SPLIT>;
    if (cudaError_t e = allow_smem(kern, done, tca_smem<D>())) return e;
    cudaError_t e = launch(kern, dim3((unsigned)plan.items, tp.splits), dim3(kTcaThreads), tca_smem<D>(), stream, pdl, tp);
    if (e != cudaSuccess) return e;
    if (tp.splits > 1) e = launch(attn_tc_join_kernel<D>, dim3((unsigned)plan.items, tp.rows / 8), dim3(256), p.seqs * sizeof(int), stream, pdl, tp);
    return e != cudaSuccess ? e : cudaGetLastError();
}

static int attn_block_shift(int block_size) {
    for (int s = 4; s <= 7; ++s)
        if (block_size == 1 << s) return s;
    return -1;
}

}  // namespace ztq

using namespace ztq;

extern "C" {

int ztq_take_error_attn() { return take_error(); }

size_t ztq_attn_q8_workspace_bytes(int tokens, int sequences, int max_new, int q_heads, int kv_heads, int head_dim) {
    if (tokens < 0 || sequences <= 0 || max_new <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return 0;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    const int sms = device_info().sms > 0 ? device_info().sms : 148, group = q_heads / kv_heads;
    const long long rows = (long long)max_new * group;
    const int nt = attn_nt(head_dim, rows, false);
    return std::max((size_t)sms * 2 * 8 * nt * (head_dim + 2) * sizeof(float),
                    std::max(tc_plan(tokens, sequences, rows, group, kv_heads, head_dim, false, sms).bytes, tc_plan(tokens, sequences, rows, group, kv_heads, head_dim, true, sms).bytes));
}

cudaError_t ztq_attn_q8(const void* q, void* y, long long q_token, long long q_head, long long y_token, long long y_head, int tokens, int q_heads,
                        const int* query_start, const int* kv_len, const int* block_table, int sequences, int table_width, int max_new, int window,
                        unsigned scale_bits, const ZtqKvCache* cache, void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream) {
    if ((tokens != 0 && (!q || !y)) || !query_start || !kv_len || !block_table || !cache || !cache->k || !cache->v || !cache->k_scale || !cache->v_scale || !workspace) return cudaErrorInvalidValue;
    const int shift = attn_block_shift(cache->block_size), dim = cache->head_dim;
    if (shift < 0 || (dim != 64 && dim != 128 && dim != 256) || cache->blocks <= 0 || cache->kv_heads <= 0) return cudaErrorInvalidValue;
    if (cache->block_stride < (long long)cache->kv_heads * cache->block_size * dim || cache->block_stride % 16) return cudaErrorInvalidValue;
    if (((uintptr_t)cache->k | (uintptr_t)cache->v | (uintptr_t)workspace) & 15) return cudaErrorInvalidValue;
    if (tokens < 0 || q_heads <= 0 || q_heads % cache->kv_heads || sequences <= 0 || sequences > kAttnMaxSeqs || table_width <= 0 || max_new <= 0 || window < 0)
        return cudaErrorInvalidValue;
    if ((long long)table_width << shift > 0x7fffffffll || (long long)max_new * (q_heads / cache->kv_heads) > 0x7fffffffll) return cudaErrorInvalidValue;
    if (flags & ~(ZTQ_X_F32 | ZTQ_Y_F32 | ZTQ_NO_PDL)) return cudaErrorInvalidValue;
    if (workspace_bytes < ztq_attn_q8_workspace_bytes(tokens, sequences, max_new, q_heads, cache->kv_heads, dim)) return cudaErrorInvalidValue;
    float scale;
    memcpy(&scale, &scale_bits, 4);
    const DeviceInfo dev = device_info();
    if (dev.major < 10) return cudaErrorNoKernelImageForDevice;
    if (tokens == 0) return cudaSuccess;
    AttnParams p = {};
    p.q = q;
    p.y = y;
    p.q_token = q_token; p.q_head = q_head; p.y_token = y_token; p.y_head = y_head;
    p.query_start = query_start;
    p.kv_len = kv_len;
    p.block_table = block_table;
    p.kc = static_cast<const int8_t*>(cache->k);
    p.vc = static_cast<const int8_t*>(cache->v);
    p.ks = cache->k_scale;
    p.vs = cache->v_scale;
    p.block_stride = cache->block_stride;
    p.parts = static_cast<float*>(workspace);
    p.seqs = sequences;
    p.tokens = tokens;
    p.max_new = max_new;
    p.q_heads = q_heads;
    p.kv_heads = cache->kv_heads;
    p.group = q_heads / cache->kv_heads;
    p.width = table_width;
    p.shift = shift;
    p.blocks = cache->blocks;
    p.window = window;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.x_f32 = (flags & ZTQ_X_F32) ? 1 : 0;
    p.y_f32 = (flags & ZTQ_Y_F32) ? 1 : 0;
    p.vec = ((uintptr_t)q & (p.x_f32 ? 15 : 7)) == 0 && q_token % 4 == 0 && q_head % 4 == 0;
    const int wide = p.y_f32 ? 4 : 8;
    p.y_wide = ((uintptr_t)y & 15) == 0 && y_token % wide == 0 && y_head % wide == 0;
    p.min_rows = 1;
    p.max_rows = 0x7fffffff;
    const bool split = p.x_f32 || p.y_f32, pdl = !(flags & ZTQ_NO_PDL);
    const int nt = attn_nt(dim, (long long)max_new * p.group, split);
    const TcPlan plan = tc_plan(tokens, sequences, (long long)max_new * p.group, p.group, p.kv_heads, dim, split, dev.sms);
    if (plan.items > 0x7fffffff) return cudaErrorInvalidValue;
    if (plan.items > 0) {
        if (!plan.all) p.min_rows = kTcMinRows + 1;              // told apart on the device, where the lengths are
        cudaError_t e = dim == 64 ? (split ? launch_tc<64, true>(p, plan, stream, pdl) : launch_tc<64, false>(p, plan, stream, pdl))
                                  : (split ? launch_tc<128, true>(p, plan, stream, pdl) : launch_tc<128, false>(p, plan, stream, pdl));
        if (e != cudaSuccess || plan.all) return e;
        p.min_rows = 1;
        p.max_rows = kTcMinRows;
    }
    return dim == 64 ? launch_dim<64>(p, nt, split, dev.sms, stream, pdl)
         : dim == 128 ? launch_dim<128>(p, nt, split, dev.sms, stream, pdl) : launch_dim<256>(p, nt, split, dev.sms, stream, pdl);
}

}  // extern "C"
