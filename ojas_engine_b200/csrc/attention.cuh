// Attention over a paged cache: what its two kernels, the joining kernel and the entry point share.
#pragma once
#include <atomic>

#include "attn.cuh"
#include "tc_util.cuh"

struct AttnArgs {
    const void *q;
    void *out;
    long long q_stride, out_stride;      // elements between tokens
    BatchArgs batch;
    float *part_o;                       // [splits][M][q_heads][dim] unnormalized sums (null: one split)
    float2 *part_ml;                     // [splits][M][q_heads] (maximum in log2 units, sum); sum < 0: the row is already in out
    uint32_t act_type;
    int q_heads, group;                  // group = query heads per key head
    int splits, split_blocks;            // key blocks per split
    int window;                          // 0: none
    bool causal;
    float scale_log2;                    // softmax scale * log2(e)
};

// A row is one (token, query head) pair; the rows of a sequence that share a key head are numbered token * group + head in
// group, and a tile is `rows` of them.  Tile t of the call belongs to the sequence found by walking the row counts.
struct RowTile {
    int seq, row0, n_rows;               // first row in the sequence, rows of the sequence (all of them)
    int token0;                          // call row of the sequence's first new token
    int pos0;                            // cache position of its first new token
    int len;                             // keys that may be read
};

// One warp, all lanes: which sequence tile `tile` (counted over all sequences) falls in.  False: behind the last one.
// Every value is clamped so that no description, however wrong, leads outside the arrays; a wrong one sets the status bit.
__device__ __forceinline__ bool find_tile(const AttnArgs &a, int tile, int rows, int lane, RowTile &t) {
    const BatchArgs &b = a.batch;
    long long before = 0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        long long first = 0, n = 0;
        if (s < b.n_seqs) {
            first = max(0, __ldg(b.cu + s));
            n = min((long long)__ldg(b.cu + s + 1), b.M) - first;
            n = n < 0 ? 0 : n;
        }
        const int tiles = (int)((n * a.group + rows - 1) / rows);
        int sum = tiles;                                          // inclusive prefix over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + sum > tile);
        if (hit) {
            const int src = __ffs(hit) - 1;
            t.seq = s0 + src;
            t.token0 = (int)__shfl_sync(0xffffffffu, first, src);
            const int tokens = (int)__shfl_sync(0xffffffffu, n, src);
            t.n_rows = tokens * a.group;
            t.row0 = (int)(tile - before - __shfl_sync(0xffffffffu, sum - tiles, src)) * rows;
            const int len = __ldg(b.len + t.seq);
            const long long room = (long long)b.table_stride * b.page_size;
            t.pos0 = len - tokens;
            t.len = (int)max(0ll, min((long long)len, room));
            if (lane == 0 && ((long long)len > room || len < tokens || tokens > b.max_rows)) atomicOr(b.status, OJAS_ST_BATCH);
            return t.row0 >= 0 && t.row0 < t.n_rows;              // (offsets out of order could overflow the count)
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

// Keys [lo, hi) that rows [row0, row1) of the tile's sequence see, taken together (empty: hi <= lo).
__device__ __forceinline__ void key_range(const AttnArgs &a, const RowTile &t, int row0, int row1, int &lo, int &hi) {
    const long long p0 = (long long)t.pos0 + row0 / a.group, p1 = (long long)t.pos0 + (row1 - 1) / a.group;
    hi = a.causal ? (int)max(0ll, min((long long)t.len, p1 + 1)) : t.len;
    lo = a.window ? (int)max(0ll, p0 - a.window + 1) : 0;
}
// The same for one row: key j is seen when lo <= j < hi.
__device__ __forceinline__ void row_range(const AttnArgs &a, const RowTile &t, int row, int &lo, int &hi) { key_range(a, t, row, row + 1, lo, hi); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Allows a kernel its dynamic shared memory, once per device (a bit each; devices from 64 on are asked every time).
template <typename K>
static cudaError_t smem_once(std::atomic<uint64_t> &ready, int device, K kernel, int bytes) {
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if (bit && (ready.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// What the planner decides for a call (attention.cu).
struct AttnPlan {
    bool tensor;                         // the tcgen05 kernel
    bool two, cluster;                   // the kernel for few rows: two terms per value; the splits are a cluster
    int rows, mt;                        // rows of a tile; MMA tiles per warp of the kernel for few rows
    long long tiles;                     // upper bound on the call's row tiles
    int splits, split_blocks, block;     // keys per block
    size_t workspace;
};
int attn_tc_launch(ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p);
