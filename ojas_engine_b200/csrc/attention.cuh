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
    int per_seq;                         // row tiles of every sequence (0: as many as its rows need)
    int window;                          // 0: none
    bool causal;
    float scale_log2;                    // softmax scale * log2(e)
};

// Keys are counted in 32 bits, and what rounds their number up to a block, or steps past the last, must not pass them.
constexpr long long ATTN_MOST_KEYS = 0x7fffff00;

// A row is one (token, query head) pair; the rows of a sequence that share a key head are numbered token * group + head in
// group, and a tile is `rows` of them.
struct RowTile {
    int seq, row0, n_rows;               // first row in the sequence, rows of the sequence (all of them)
    int token0;                          // call row of the sequence's first new token
    int pos0;                            // cache position of its first new token
    int len;                             // keys that may be read
};

// First row and number of rows of sequence s, clamped to the call, and its end as given.  False: its offsets lead outside the call, or back.
__device__ __forceinline__ bool seq_rows(const BatchArgs &b, int s, int &first, int &n, int &end) {
    const int start = __ldg(b.cu + s);
    end = __ldg(b.cu + s + 1);
    first = max(0, start);
    n = (int)max(0ll, min((long long)end, b.M) - first);
    return seq_in_call(start, end, b.M);
}

// One warp, all lanes: which rows tile `tile` of the call is.  With per_seq > 0 every sequence has that many tiles, used or not; else
// tiles are counted over the sequences' rows, 128 sequences at a time.  False: no such rows.  Every value is clamped so that no
// description, however wrong, leads outside the arrays; a wrong one sets the status bit.  (Every sequence is looked at by some tile: with
// per_seq by its own; else the offsets in front of the first wrong ones hold fewer tiles than the call has, so its last tile looks past them.)
__device__ __forceinline__ bool find_tile(const AttnArgs &a, int tile, int rows, int lane, RowTile &t) {
    const BatchArgs &b = a.batch;
    int first = 0, n = 0, end = 0;
    bool in_call = true;
    long long before = 0;                                         // tiles of the sequences in front
    if (a.per_seq > 0) {
        t.seq = tile / a.per_seq;
        if (t.seq >= b.n_seqs) return false;
        before = (long long)t.seq * a.per_seq;
        in_call = seq_rows(b, t.seq, first, n, end);
        if (!in_call && lane == 0) atomicOr(b.status, OJAS_ST_BATCH);
    } else {
        bool found = false;
        for (int s0 = 0; s0 < b.n_seqs && !found; s0 += 128) {
            int start[4], count[4], tiles[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int s = s0 + lane * 4 + i;
                start[i] = count[i] = 0;
                if (s < b.n_seqs && !seq_rows(b, s, start[i], count[i], end)) in_call = false;
                tiles[i] = (int)(((long long)count[i] * a.group + rows - 1) / rows);
                sum += tiles[i];
            }
            int upto = sum;                                       // inclusive prefix over the lanes
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + upto > tile);
            if (hit) {
                const int src = __ffs(hit) - 1;
                long long at = before + upto - sum;               // the lane's own sequences
                int which = 0;
#pragma unroll
                for (int i = 0; i < 3; i++)
                    if (which == i && at + tiles[i] <= tile) { at += tiles[i]; which = i + 1; }
                t.seq = s0 + src * 4 + __shfl_sync(0xffffffffu, which, src);
                first = __shfl_sync(0xffffffffu, which == 0 ? start[0] : which == 1 ? start[1] : which == 2 ? start[2] : start[3], src);
                n = __shfl_sync(0xffffffffu, which == 0 ? count[0] : which == 1 ? count[1] : which == 2 ? count[2] : count[3], src);
                before = __shfl_sync(0xffffffffu, at, src);
                found = true;
            } else {
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (!in_call) atomicOr(b.status, OJAS_ST_BATCH);
        if (!found) return false;
        end = __ldg(b.cu + t.seq + 1);
    }
    t.token0 = first;
    t.n_rows = n * a.group;
    t.row0 = (int)(tile - before) * rows;
    const int len = __ldg(b.len + t.seq);
    const long long room = min((long long)b.table_stride * b.page_size, ATTN_MOST_KEYS);
    t.pos0 = (int)max(-0x40000000ll, min(0x7fffffffll, (long long)len - end + first));   // where the append puts the row, whatever lies outside the call
    t.len = (int)max(0ll, min((long long)len, room));
    if (lane == 0 && n > 0 && ((long long)len > room || len < n || n > b.max_rows)) atomicOr(b.status, OJAS_ST_BATCH);
    return t.row0 >= 0 && t.row0 < t.n_rows;                      // (offsets out of order could overflow the count)
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

// Allows a kernel its dynamic shared memory, and clusters of more than eight CTAs, once per device (two bits each; devices from
// 32 on are asked every time).
template <typename K>
static cudaError_t smem_once(std::atomic<uint64_t> &ready, int device, K kernel, int bytes, bool large_clusters = false) {
    const uint64_t bit = device < 32 ? 1ull << (2 * device) : 0ull, want = large_clusters ? 3 * bit : bit;
    if (bit && (ready.load(std::memory_order_relaxed) & want) == want) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && large_clusters) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) ready.fetch_or(want, std::memory_order_relaxed);
    return e;
}

// What the planner decides for a call (attention.cu).
struct AttnPlan {
    bool tensor;                         // the tcgen05 kernel
    bool two, cluster;                   // the kernel for few rows: two terms per value; the splits are a cluster
    int rows, mt;                        // rows of a tile; MMA tiles per warp of the kernel for few rows
    long long tiles;                     // upper bound on the call's row tiles
    int per_seq;                         // see AttnArgs
    int splits, split_blocks, block;     // keys per block
    size_t workspace;
};
int attn_tc_launch(ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p);
