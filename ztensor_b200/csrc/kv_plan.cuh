// kv_plan.cuh -- the plan of one serving step, built on the GPU from the sequences' lengths.
//
// With c = tokens cached, a = tokens of this step, bs = tokens per block:
//   have = ceil(c / bs),  want = ceil((c + a) / bs),  ask = want - have,
//   first row of a sequence = exclusive prefix sum of a,  its new blocks = ring[(head + prefix of ask + k) mod pool],
//   slot of its i-th token = block of position c + i times bs + (c + i) mod bs.
// Everything is integer arithmetic on two prefix sums over the sequences, so the result does not depend on the launch.
//
// One cluster of CTAs: each holds the sums of all sequences in its own shared memory (recomputing them costs less than
// passing them on) and writes its share of the rows and of the block table.  All inputs that an output may alias are
// read before the cluster barrier and all outputs written after it.  A step moves a few KB to a few hundred KB, so what
// bounds it is the chain launch -> lengths -> sums -> rows -> store: 4.5 us for 8 sequences, 8.7 for 1024 with 24 prompts and 9
// that end (10.3 when the blocks they give back moved one load at a time).
#pragma once

#include "ztq_common.cuh"

namespace ztq {

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxSeqs = 4096;

struct PlanParams {
    const int* ctx_len;
    const int* new_len;
    int* block_table;
    int* ring;
    const int* ring_state;
    int* ring_state_out;
    int* next_len;
    int* kv_len;
    int* query_start;
    int* positions;
    int* slots;
    int* status;
    int seqs, width, shift, pool, rows;      // shift: log2 of the block size
};

enum : int { PLAN_OK = 0, PLAN_POOL = 1, PLAN_TABLE = 2, PLAN_ROWS = 3, PLAN_LENGTH = 4 };

struct PlanSeq {          // what a sequence's rows and blocks are computed from
    int ctx, first, have, want, base, flags;          // flags: status | kind << 4
};

__device__ __forceinline__ long long plan_warp_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Inclusive prefix sum over the block's threads; `total` is the sum.  `part`: 33 words of shared memory.
__device__ __forceinline__ long long plan_block_scan(long long v, long long* part, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    v = plan_warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) part[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const long long s = plan_warp_scan(lane < warps ? part[lane] : 0, lane);
        __syncwarp();
        part[lane] = s;
    }
    __syncthreads();
    total = part[warps - 1];
    return v + (warp ? part[warp - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanParams p) {
    extern __shared__ PlanSeq seq[];                 // seqs entries, then seqs + 1 first rows
    __shared__ long long part[32];
    __shared__ int s_taken;
    int* first = reinterpret_cast<int*>(seq + p.seqs);
    const int tid = threadIdx.x, bs = 1 << p.shift;
    const int rank = blockIdx.x, ranks = gridDim.x;

    grid_dep_launch();
    grid_dep_wait();
    if (tid == 0) s_taken = 0;
    const int head = (int)((unsigned)p.ring_state[0] % (unsigned)p.pool);
    const int count = min(max(p.ring_state[1], 0), p.pool);

    // sums over the sequences, blockDim.x of them at a time
    long long rows_before = 0, asked_before = 0, given_before = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += blockDim.x) {
        const int b = b0 + tid;
        long long ctx = 0, add = 0;
        bool bad = false, gone = false;
        if (b < p.seqs) {
            ctx = p.ctx_len[b];
            const int n = p.new_len[b];
            bad = ctx < 0 || n < -1 || ((ctx + bs - 1) >> p.shift) > p.width;
            gone = !bad && n == -1;
            add = bad || n < 0 ? 0 : n;
        }
        long long total;
        const long long end = rows_before + plan_block_scan(add, part, total);
        rows_before += total;
        const long long have = ctx > 0 ? (ctx + bs - 1) >> p.shift : 0, want = ctx + add > 0 ? (ctx + add + bs - 1) >> p.shift : 0;
        int status = bad ? PLAN_LENGTH : PLAN_OK;
        if (add > 0) status = end > p.rows ? PLAN_ROWS : want > p.width ? PLAN_TABLE : PLAN_OK;
        const long long ask = add > 0 && status == PLAN_OK ? want - have : 0;
        const long long upto = asked_before + plan_block_scan(ask, part, total);
        asked_before += total;
        if (ask > 0 && upto > count) status = PLAN_POOL;
        const long long give = gone ? have : 0;
        const long long given = given_before + plan_block_scan(give, part, total);
        given_before += total;
        if (b < p.seqs) {
            const bool fresh = ask > 0 && status == PLAN_OK;
            seq[b] = PlanSeq{(int)ctx, (int)min(end - add, (long long)p.rows), bad ? 0 : (int)have, fresh ? (int)want : bad ? 0 : (int)have,
                             gone ? (int)min(given - give, (long long)p.pool) : (int)min(upto - ask, (long long)p.pool), status | (gone ? 16 : 0)};
            first[b + 1] = (int)min(end, (long long)p.rows);
            if (fresh) atomicMax(&s_taken, (int)upto);
        }
    }
    if (tid == 0) first[0] = 0;
    const int released = (int)min(given_before, (long long)(p.pool - count));
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");

    auto wrap = [&](int i) { return i >= p.pool ? i - p.pool : i; };
    // per sequence: lengths and status
    const int stride = ranks * blockDim.x, at = rank * blockDim.x + tid;
    for (int b = at; b < p.seqs; b += stride) {
        const PlanSeq q = seq[b];
        const int status = q.flags & 15;
        const bool gone = q.flags & 16;
        const int n = first[b + 1] - q.first;        // the sequence's rows (all of them unless the rows ran out)
        p.status[b] = status;
        p.kv_len[b] = status == PLAN_OK && !gone ? q.ctx + n : 0;
        p.next_len[b] = gone ? 0 : status == PLAN_OK ? q.ctx + n : q.ctx;
        p.query_start[b + 1] = first[b + 1];
    }
    if (at == 0) {
        p.query_start[0] = 0;
        p.ring_state_out[0] = (int)(((unsigned)head + (unsigned)s_taken) % (unsigned)p.pool);
        p.ring_state_out[1] = count - s_taken + released;
    }
    // blocks: a warp per sequence
    const int lane = tid & 31, warps = ranks * (blockDim.x >> 5);
    for (int b = rank * (blockDim.x >> 5) + (tid >> 5); b < p.seqs; b += warps) {
        const PlanSeq q = seq[b];
        int* row = p.block_table + (long long)b * p.width;
        // both indices stay below twice the pool: new blocks are among `count`, released ones among the rest
#pragma unroll 4
        for (int k = q.have + lane; k < q.want; k += 32) row[k] = p.ring[wrap(head + q.base + (k - q.have))];
        if (q.flags & 16) {
            const int n = min(q.have, released - q.base);
            for (int k = lane; k < n; k += 4 * 32) {             // four loads on their way at a time
                int block[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k + 32 * i < n) block[i] = row[k + 32 * i];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k + 32 * i < n) p.ring[wrap(wrap(head + count) + q.base + k + 32 * i)] = block[i];
            }
        }
    }
    // rows
    const int live = first[p.seqs];
    for (int t = at; t < p.rows; t += stride) {
        int pos = 0, slot = -1;
        if (t < live) {
            int lo = 0, hi = p.seqs - 1;             // the sequence whose rows hold t: smallest b with first[b + 1] > t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (first[mid + 1] > t) hi = mid; else lo = mid + 1;
            }
            const PlanSeq q = seq[lo];
            pos = (int)((unsigned)q.ctx + (unsigned)(t - q.first));
            if ((q.flags & 15) == PLAN_OK) {
                const int k = pos >> p.shift;
                const int block = k < q.have ? p.block_table[(long long)lo * p.width + k]
                                             : p.ring[wrap(head + q.base + (k - q.have))];
                if (block >= 0 && block < p.pool) slot = (block << p.shift) + (pos & (bs - 1));
            }
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
}

}  // namespace ztq
