// Attention of new tokens over a paged cache:
//     out[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[t, h] . k_j - m),   j over the keys that row (t, h) sees,
// one pass over the keys with the running maximum m and sum of each row (a row that sees nothing gives 0).  This file holds the
// kernel for few rows per key head (decoding, checking a few drafted tokens), the joining of split rows, and the entry point;
// attention_tc.cu the tcgen05 kernel for more rows.
//
// Few rows are bound by the bytes of K and V (HBM): rows * 4 flops per key byte are far below what even the warp-level MMA
// gives.  A CTA takes one tile of rows of one key head and a range of keys, in blocks of 64 that a producer warp's tensor copies bring
// straight from the pages into a ring (128-byte swizzle; issued by one of the working warps between its own blocks they cost a
// third of the rate).  Four warps take 16 keys of each block; each keeps its own running maximum and sum, and they are joined at the end.
//
// mma.m16n8k16 has 16 rows.  TWO: a tile row takes two of them, its HIGH and LOW halves: q = hi + lo in the cache's type sits in rows
// g and g + 8 of the A operand, one instruction forms hi.k and lo.k, and the score is their sum; probabilities go into the second
// product the same way.  f32 activations over an f16 cache so keep 22 bits through both products, over a bf16 cache 16 (a
// bf16 term has 8), and up to eight rows this costs nothing, so 16-bit activations take it there too.  Otherwise 16-bit
// activations use all 16 rows and round the probabilities once.  f32 rows are scaled by a power of two first so that neither term
// leaves f16's range; probabilities are kept scaled by 2^8 for the same reason.
//
// Keys are split over CTAs where there are few tiles.  Up to 16 splits that all fit on the GPU at once form a cluster and join
// through each other's shared memory (one short sequence: 9.9 -> 7.2 us); otherwise they write their sums to the workspace and a second
// kernel joins them (CTAs of a cluster hold their places until the last of them is there: 64 ragged sequences in four
// splits take 272 us as clusters, 186 us this way).
#include "attention.cuh"

// ---------------------------------------------------------------------------- few rows: warp-level MMA
constexpr int AR_KEYS = 64;                                  // keys of a block
constexpr int AR_WARPS = 4, AR_THREADS = (AR_WARPS + 1) * 32;   // consumer warps; and the producer
constexpr int AR_STAT_BYTES = 256 + AR_WARPS * 32 * 8 + 32 * 8;   // barriers; per warp and row (maximum, sum); per row the same
constexpr int AR_CLUSTER = 16;                               // most splits that are a cluster (more than 8 have to be asked for; see cluster_limit)
__host__ __device__ constexpr int ar_stage_bytes(int dim) { return 2 * AR_KEYS * dim * 2; }
// 96 KB of blocks in flight per CTA, two CTAs per SM (dim 256: three 64 KB blocks, one CTA): HBM needs about 44 KB per SM and
// microsecond of latency.
__host__ __device__ constexpr int ar_stages(int dim) { return dim == 64 ? 6 : 3; }
__host__ __device__ constexpr int ar_smem(int dim) { return ar_stages(dim) * ar_stage_bytes(dim) + AR_STAT_BYTES + 1024; }
constexpr float AR_SHIFT = 8.0f, AR_SLACK = 7.0f;            // p <= 2^(SHIFT + SLACK) < 65504; the maximum may lag by SLACK

template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// Address of element (row, col) of a block in shared memory: slabs of 64 columns, rows of 128 bytes, 16-byte pieces swizzled by the
// row's low three bits (what the tensor copy writes).
__device__ __forceinline__ uint32_t block_addr(uint32_t base, int row, int col) {
    return base + (uint32_t)((col >> 6) * (AR_KEYS * 128) + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4));
}
// v = hi + lo with both of the 16-bit type, two values packed.
template <bool BF>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = pack_half(a, b, BF);
    const float2 h = unpack_half(hi, BF);
    lo = pack_half(a - h.x, b - h.y, BF);
}

__device__ __forceinline__ uint32_t cluster_addr(uint32_t smem_addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A tile of the call is MT * (TWO ? 8 : 16) rows.
template <int D, bool BF, bool TWO, int MT>
__global__ void __launch_bounds__(AR_THREADS, MT == 2 || D == 256 ? 1 : 2) attn_rows_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                                         const __grid_constant__ CUtensorMap map_v, const AttnArgs a, int box_rows) {
    constexpr int STAGES = ar_stages(D), STAGE = ar_stage_bytes(D), HALF = STAGE / 2, NT = D / 8;
    constexpr int R = TWO ? 1 : 2, ROWS = MT * 8 * R;        // rows a lane works on per MMA tile; rows of the tile
    extern __shared__ unsigned char ar_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)ar_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + STAGES * STAGE), *empty = full + STAGES;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(empty + STAGES);
    float2 *stats = reinterpret_cast<float2 *>(smem + STAGES * STAGE + 256);      // [AR_WARPS][ROWS] (maximum, sum)
    float2 *joined = stats + AR_WARPS * 32;                                       // [ROWS] of the CTA
    static_assert(AR_WARPS * ROWS * D * 4 <= STAGES * STAGE && ROWS <= 32, "the warps' sums meet where the ring was");
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, kvh = blockIdx.y, split = blockIdx.z;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], AR_WARPS); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_v) : "memory");
    }
    grid_launch_dependents();
    grid_dependency_wait();                                  // q, the cache and the batch come from the kernels before this one
    __syncthreads();
    // What follows is the same in every thread of a cluster up to `alone`: the CTAs of a cluster leave together or not at all.
    RowTile t;
    if (!find_tile(a, blockIdx.x, ROWS, lane, t)) return;    // the same answer in every warp
    const int rows = min(ROWS, t.n_rows - t.row0);
    int lo, hi;
    key_range(a, t, t.row0, t.row0 + rows, lo, hi);
    const int blk_all0 = lo / AR_KEYS, blk_all1 = hi > lo ? (hi + AR_KEYS - 1) / AR_KEYS : blk_all0;
    // (the last split takes all that is left: the result does not depend on the bounds the split was planned with)
    const bool alone = a.splits == 1 || blk_all1 - blk_all0 <= a.split_blocks;   // this tile has one split: straight to out
    if (alone && split > 0) return;
    const int blk0 = min(blk_all1, blk_all0 + split * a.split_blocks);
    const int blk1 = split == a.splits - 1 ? blk_all1 : min(blk_all1, blk0 + a.split_blocks);

    if (warp == AR_WARPS) {
        // ---------------- producer: lane = one box (64 values x box_rows tokens) of K or V; pages are looked up a block ahead
        const int per_slab = AR_KEYS / box_rows, boxes = 2 * per_slab * (D / 64);
        const int part = lane % per_slab, slab = lane / per_slab % (D / 64), page_size = a.batch.page_size;
        const bool is_v = lane >= boxes / 2;
        const int *table = a.batch.table + (long long)t.seq * a.batch.table_stride;
        auto wanted = [&](int key) { return lane < boxes && key < hi && key + box_rows > lo; };
        int key = blk0 * AR_KEYS + part * box_rows, entry = key / page_size, slot = key - entry * page_size;
        const int step_entry = AR_KEYS / page_size, step_slot = AR_KEYS - step_entry * page_size;
        int next_page = blk0 < blk1 && wanted(key) ? __ldg(table + entry) : -1;
        uint32_t phase = 1;
        int s = 0;
        for (int blk = blk0; blk < blk1; blk++) {
            const bool want = wanted(key);
            const int at = slot;
            int page = next_page;
            key += AR_KEYS;
            entry += step_entry;
            slot += step_slot;
            if (slot >= page_size) { slot -= page_size; entry++; }
            next_page = blk + 1 < blk1 && wanted(key) ? __ldg(table + entry) : -1;
            if (!mbar_wait_warp(&empty[s], phase, abort_flag, a.batch.status, OJAS_ST_ATTN_WAIT)) break;
            if (want && (page < 0 || page >= a.batch.pages)) { atomicOr(a.batch.status, OJAS_ST_BATCH); page = a.batch.pages; }   // reads as zeros
            const int n = __popc(__ballot_sync(0xffffffffu, want));
            if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(n * box_rows * 128));
            __syncwarp();
            if (want)
                tma_load_4d(smem + s * STAGE + (is_v ? HALF : 0) + slab * (AR_KEYS * 128) + part * box_rows * 128, is_v ? &map_v : &map_k, slab * 64, at, kvh, page, &full[s]);
            if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
    }
    const int g = lane >> 2, q4 = lane & 3;
    float o[MT][NT][4];
    float m[MT][R], l[MT][R], factor[MT][R];                 // factor: score -> log2 units
    int see_lo[MT][R], see_hi[MT][R];
    if (warp < AR_WARPS) {
    // ---------------- q: this lane's pairs of its rows
    uint32_t qf[MT][D / 16][4];
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int n = 0; n < NT; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int in_tile = i * 8 * R + r * 8 + g, row = t.row0 + in_tile;
            const bool live = in_tile < rows;
            m[i][r] = -INFINITY; l[i][r] = 0.0f;
            see_lo[i][r] = see_hi[i][r] = 0;
            factor[i][r] = a.scale_log2;
            const long long at = live ? (long long)(t.token0 + row / a.group) * a.q_stride + (long long)(kvh * a.group + row % a.group) * D : 0;
            if (live) row_range(a, t, row, see_lo[i][r], see_hi[i][r]);
            if (TWO && a.act_type == OJAS_B200_F32) {
                const float *q = static_cast<const float *>(a.q) + at;
                float2 v[D / 8];
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < D / 8; k++) {
                    v[k] = live ? *reinterpret_cast<const float2 *>(q + k * 8 + 2 * q4) : make_float2(0.f, 0.f);
                    top = fmaxf(top, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^e in (top/2, top]: the row over 2^e is below 2 (zero, infinite and subnormal rows stay as they are)
                const uint32_t e = __float_as_uint(top) & 0x7f800000u;
                const bool scalable = e > 0x01000000u && e < 0x7e000000u;
                const float up = scalable ? __uint_as_float(e) : 1.0f, down = scalable ? __uint_as_float(0x7f000000u - e) : 1.0f;
                factor[i][r] *= up;
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    split_pair<BF>(v[2 * k].x * down, v[2 * k].y * down, qf[i][k][0], qf[i][k][1]);
                    split_pair<BF>(v[2 * k + 1].x * down, v[2 * k + 1].y * down, qf[i][k][2], qf[i][k][3]);
                }
            } else {
                const uint32_t *q = reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(a.q) + at);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    qf[i][k][r] = live ? q[k * 8 + q4] : 0u;
                    qf[i][k][2 + r] = live ? q[k * 8 + 4 + q4] : 0u;
                    if (TWO) qf[i][k][1] = qf[i][k][3] = 0u;
                }
            }
        }
    }
    const int mi = lane >> 3, mr = lane & 7;                 // ldmatrix: which 8x8 matrix this lane addresses, and its row
    uint32_t phase = 0;
    int s = 0;
    for (int blk = blk0; blk < blk1; blk++) {
        if (!mbar_wait_warp(&full[s], phase, abort_flag, a.batch.status, OJAS_ST_ATTN_WAIT)) break;
        const int key0 = blk * AR_KEYS + warp * 16;
        const uint32_t kb = smem_u32(smem + s * STAGE), vb = kb + HALF;
        if (key0 < hi && key0 + 16 > lo) {
            if (key0 < lo || key0 + 16 > hi) {
                // what lies behind the sequence or was not copied may be anything, and 0 * NaN is NaN: this warp's keys outside
                // [lo, hi) get zeros for values
                for (int i = lane; i < 16 * (D / 8); i += 32) {
                    const int r = i / (D / 8), c = i % (D / 8) * 8;
                    if (key0 + r < lo || key0 + r >= hi)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(block_addr(vb, warp * 16 + r, c)), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy into this stage
                __syncwarp();
            }
            float sc[MT][2][4];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int n = 0; n < 2; n++) sc[i][n][0] = sc[i][n][1] = sc[i][n][2] = sc[i][n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                uint32_t b[4];
                ldsm4(b, block_addr(kb, warp * 16 + (mi >> 1) * 8 + mr, k * 16 + (mi & 1) * 8));
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    mma16816<BF>(sc[i][0], qf[i][k], b[0], b[1]);
                    mma16816<BF>(sc[i][1], qf[i][k], b[2], b[3]);
                }
            }
            uint32_t pf[MT][4];
#pragma unroll
            for (int i = 0; i < MT; i++) {
                float x[R][4];                               // a row's keys key0 + 2 q4 + {0, 1, 8, 9}
                bool grow = false;
                float top[R];
#pragma unroll
                for (int r = 0; r < R; r++) {
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int key = key0 + n * 8 + 2 * q4 + e;
                            const float v = (TWO ? sc[i][n][e] + sc[i][n][e + 2] : sc[i][n][e + 2 * r]) * factor[i][r];
                            x[r][2 * n + e] = key >= see_lo[i][r] && key < see_hi[i][r] ? v : -INFINITY;
                        }
                    top[r] = fmaxf(fmaxf(x[r][0], x[r][1]), fmaxf(x[r][2], x[r][3]));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    grow |= top[r] > m[i][r] + AR_SLACK;     // (-inf + slack = -inf: the first seen key always raises it)
                }
                if (__any_sync(0xffffffffu, grow)) {
                    float f[2];
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const float mn = top[r] > m[i][r] + AR_SLACK ? top[r] : m[i][r];
                        f[r] = mn == m[i][r] ? 1.0f : exp2_fast(m[i][r] - mn);
                        m[i][r] = mn;
                        l[i][r] *= f[r];
                    }
                    if (TWO) f[1] = f[0];
#pragma unroll
                    for (int n = 0; n < NT; n++) { o[i][n][0] *= f[0]; o[i][n][1] *= f[0]; o[i][n][2] *= f[1]; o[i][n][3] *= f[1]; }
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float off = m[i][r] == -INFINITY ? 0.0f : m[i][r] - AR_SHIFT;
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) { p[e] = exp2_fast(x[r][e] - off); l[i][r] += p[e]; }
                    if (TWO) {
                        split_pair<BF>(p[0], p[1], pf[i][0], pf[i][1]);
                        split_pair<BF>(p[2], p[3], pf[i][2], pf[i][3]);
                    } else {
                        pf[i][r] = pack_half(p[0], p[1], BF);
                        pf[i][2 + r] = pack_half(p[2], p[3], BF);
                    }
                }
            }
#pragma unroll
            for (int n2 = 0; n2 < D / 16; n2++) {
                uint32_t b[4];
                ldsm4_trans(b, block_addr(vb, warp * 16 + (mi & 1) * 8 + mr, n2 * 16 + (mi >> 1) * 8));
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    mma16816<BF>(o[i][2 * n2], pf[i], b[0], b[1]);
                    mma16816<BF>(o[i][2 * n2 + 1], pf[i], b[2], b[3]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == STAGES) { s = 0; phase ^= 1u; }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int r = 0; r < R; r++) {
            l[i][r] += __shfl_xor_sync(0xffffffffu, l[i][r], 1);
            l[i][r] += __shfl_xor_sync(0xffffffffu, l[i][r], 2);
            if (l[i][r] != l[i][r] && m[i][r] == -INFINITY) m[i][r] = 0.0f;       // nothing but NaN was seen: that is not "no key"
            if (q4 == 0) stats[warp * ROWS + i * 8 * R + r * 8 + g] = make_float2(m[i][r], l[i][r]);
        }
    }
    __syncthreads();                                         // the ring is free: every copy that was issued has been waited for
    if (*abort_flag) {                                       // copies still in flight get a bounded time to land
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    // ---------------- the warps' sums, each scaled to the row's maximum, meet in shared memory
    float *sums = reinterpret_cast<float *>(smem);           // [AR_WARPS][ROWS][D]
    if (warp < AR_WARPS) {
#pragma unroll
    for (int i = 0; i < MT; i++) {
        float f[2];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int row = i * 8 * R + r * 8 + g;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < AR_WARPS; w++) top = fmaxf(top, stats[w * ROWS + row].x);
            f[r] = m[i][r] == -INFINITY ? 0.0f : m[i][r] == top ? 1.0f : exp2_fast(m[i][r] - top);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float *to = sums + (warp * ROWS + i * 8 * R + g) * D + n * 8 + 2 * q4;
            if (TWO) *reinterpret_cast<float2 *>(to) = make_float2((o[i][n][0] + o[i][n][2]) * f[0], (o[i][n][1] + o[i][n][3]) * f[0]);
            else {
                *reinterpret_cast<float2 *>(to) = make_float2(o[i][n][0] * f[0], o[i][n][1] * f[0]);
                *reinterpret_cast<float2 *>(to + 8 * D) = make_float2(o[i][n][2] * f[1], o[i][n][3] * f[1]);
            }
        }
    }
    }
    __syncthreads();
    const bool cluster = !alone && a.part_ml == nullptr;     // splits join through shared memory
    for (int i = threadIdx.x; i < rows * (D / 4); i += AR_THREADS) {
        const int r = i / (D / 4), c = i % (D / 4) * 4, row = t.row0 + r;
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < AR_WARPS; w++) top = fmaxf(top, stats[w * ROWS + r].x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < AR_WARPS; w++) {
            const float2 st = stats[w * ROWS + r];
            total += st.x == -INFINITY ? 0.0f : st.x == top ? st.y : st.y * exp2_fast(st.x - top);
            const float4 x = *reinterpret_cast<const float4 *>(sums + (w * ROWS + r) * D + c);
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        const long long token = t.token0 + row / a.group;
        const int head = kvh * a.group + row % a.group;
        if (alone) {
            const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
            store_elem4(a.out, a.act_type, token * a.out_stride + (long long)head * D + c, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            if (a.part_ml && c == 0) a.part_ml[token * a.q_heads + head] = make_float2(0.0f, -1.0f);
        } else if (cluster) {
            *reinterpret_cast<float4 *>(sums + r * D + c) = v;                    // (only this thread reads and writes this piece)
            if (c == 0) joined[r] = make_float2(top, total);
        } else {
            const long long slot = ((long long)split * a.batch.M + token) * a.q_heads + head;
            if (blk1 > blk0) *reinterpret_cast<float4 *>(a.part_o + slot * D + c) = v;
            if (c == 0) a.part_ml[slot] = make_float2(top, total);
        }
    }
    if (!cluster) return;
    // ---------------- the splits' sums: each CTA of the cluster joins a part of the rows' pieces
    cluster_sync();
    const uint32_t sums_at = smem_u32(sums), joined_at = smem_u32(joined);
    for (int i = split * AR_THREADS + (int)threadIdx.x; i < rows * (D / 4); i += a.splits * AR_THREADS) {
        const int r = i / (D / 4), c = i % (D / 4) * 4, row = t.row0 + r;
        float2 ml[AR_CLUSTER];
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int k = 0; k < AR_CLUSTER; k++) {
            ml[k] = k < a.splits ? cluster_load2(cluster_addr(joined_at + r * 8, k)) : make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, ml[k].x);
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < AR_CLUSTER; k++) {
            if (ml[k].x == -INFINITY) continue;              // saw no key of this row
            const float f = ml[k].x == top ? 1.0f : exp2_fast(ml[k].x - top);
            const float4 x = cluster_load4(cluster_addr(sums_at + (uint32_t)(r * D + c) * 4, k));
            total += ml[k].y * f;
            v.x += x.x * f; v.y += x.y * f; v.z += x.z * f; v.w += x.w * f;
        }
        const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
        store_elem4(a.out, a.act_type, (t.token0 + row / a.group) * a.out_stride + (long long)(kvh * a.group + row % a.group) * D + c,
                    make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
    cluster_sync();                                          // nobody leaves while its sums are being read
}

// ---------------------------------------------------------------------------- joining the splits
// One warp per (token, head): the splits' sums, each scaled to the row's maximum, over the total.  Rows that a kernel finished
// itself, and rows of no sequence, are left alone.
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = a.batch.M * a.q_heads;
    if (row >= rows) return;
    const long long token = row / a.q_heads;
    // lane s holds split s's maximum and sum (further splits: a second round), then its weight
    constexpr int V = D / 32;                                // values per lane
    float acc[V], total = 0.0f, top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    float2 ml = lane < a.splits ? a.part_ml[(long long)lane * rows + row] : make_float2(-INFINITY, 0.0f);
    const bool mine = token >= __ldg(a.batch.cu) && token < __ldg(a.batch.cu + a.batch.n_seqs);
    if (!mine || __shfl_sync(0xffffffffu, ml.y, 0) < 0.0f) return;
    for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, s == lane ? ml.x : a.part_ml[(long long)s * rows + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int s0 = 0; s0 < a.splits; s0 += 32) {
        if (s0 > 0) ml = s0 + lane < a.splits ? a.part_ml[(long long)(s0 + lane) * rows + row] : make_float2(-INFINITY, 0.0f);
        const float weight = ml.x == -INFINITY ? 0.0f : ml.x == top ? 1.0f : exp2_fast(ml.x - top);
        total += warp_sum(ml.x == -INFINITY ? 0.0f : ml.y * weight);
        const unsigned seen = __ballot_sync(0xffffffffu, ml.x != -INFINITY);      // the others saw no key of this row and may not have written sums
        const int n = min(32, a.splits - s0);
#pragma unroll 4
        for (int s = 0; s < n; s++) {
            const float f = __shfl_sync(0xffffffffu, weight, s);
            const float *o = a.part_o + ((long long)(s0 + s) * rows + row) * D + lane * V;
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 x = seen >> s & 1u ? *reinterpret_cast<const float2 *>(o + i) : make_float2(0.f, 0.f);
                acc[i] += x.x * f;
                acc[i + 1] += x.y * f;
            }
        }
    }
    const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
    const long long at = token * a.out_stride + (row - token * a.q_heads) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        if (a.act_type == OJAS_B200_F32) *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + i) = make_float2(acc[i] * inv, acc[i + 1] * inv);
        else *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + at + i) = pack_half(acc[i] * inv, acc[i + 1] * inv, a.act_type == OJAS_B200_BF16);
    }
}

// ---------------------------------------------------------------------------- plan
constexpr float LOG2_E = 1.4426950408889634f;
static int attn_shape_check(uint32_t cache_type, size_t page_size, size_t kv_heads, size_t dim, uint32_t act_type, size_t q_heads, size_t M, size_t max_rows,
                            size_t max_len, char *err, size_t errlen) {
    auto no = [&](int code, const char *why) { if (err && errlen) snprintf(err, errlen, "attention: %s", why); return code; };
    if (dim != 64 && dim != 128 && dim != 256) return no(OJAS_B200_E_UNSUPPORTED, "the head size must be 64, 128 or 256");
    if (cache_type != OJAS_B200_F16 && cache_type != OJAS_B200_BF16) return no(OJAS_B200_E_ARG, "a cache holds f16 or bf16");
    if (act_type != OJAS_B200_F32 && act_type != cache_type) return no(OJAS_B200_E_UNSUPPORTED, "activations must be f32 or the cache's type");
    if (page_size == 0 || page_size % 16) return no(OJAS_B200_E_UNSUPPORTED, "the page size must be a multiple of 16 tokens");
    if (kv_heads == 0 || kv_heads > 65535 || q_heads == 0 || q_heads > 65536 || q_heads % kv_heads) return no(OJAS_B200_E_ARG, "query heads must be a multiple of the cache's heads");
    if (M > 0x3fffffffull || max_rows > 0x3fffffffull || max_len > (size_t)ATTN_MOST_KEYS || M * (q_heads / kv_heads) > 0x3fffffffull)
        return no(OJAS_B200_E_LIMIT, "too many rows or keys");
    return 0;
}

// The most splits of the kernel for few rows that the device can place as one cluster: up to 16 where two CTAs share an SM, up to 8 where
// one has it (sixteen would need most of a GPC at once); fewer, or none (1), where its GPCs have fewer free SMs, as a partitioned device may.  Asked
// once per device, of the instance that needs most.
template <int D>
static int placeable(int device, int most) {
    static std::atomic<uint64_t> ready{0};
    int fit = 0;
    while (most > 1) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = (unsigned)most;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1, 1, (unsigned)most); cfg.blockDim = dim3(AR_THREADS); cfg.dynamicSmemBytes = ar_smem(D);
        cfg.attrs = attr; cfg.numAttrs = 1;
        if (smem_once(ready, device, attn_rows_kernel<D, false, true, 1>, ar_smem(D), most > 8) == cudaSuccess &&
            cudaOccupancyMaxActiveClusters(&fit, attn_rows_kernel<D, false, true, 1>, &cfg) == cudaSuccess && fit > 0) break;
        cudaGetLastError();                                  // a refusal is an answer
        most /= 2;
    }
    return most;
}
static int cluster_limit(int device, bool pairs) {
    static std::atomic<int> known[2][32];                    // 0: not asked yet
    int limit = device < 32 ? known[pairs][device].load(std::memory_order_relaxed) : 0;
    if (limit == 0) {
        DeviceGuard guard(device);
        limit = pairs ? placeable<128>(device, AR_CLUSTER) : placeable<256>(device, AR_CLUSTER / 2);
        if (device < 32) known[pairs][device].store(limit, std::memory_order_relaxed);
    }
    return limit;
}

// Which kernel, and how far the keys are split so that few rows still use every SM.
static AttnPlan attn_plan(const ojas_b200_ctx *ctx, size_t n_seqs, size_t M, size_t max_rows, size_t max_len, size_t q_heads, size_t kv_heads, size_t dim, size_t window, bool f32) {
    AttnPlan p{};
    const size_t group = q_heads / kv_heads, bound = (max_rows < M ? max_rows : M) * group;
    p.two = f32 || bound <= 8;
    const size_t unit = p.two ? 8 : 16;                      // rows of an MMA tile
    // More rows than this kernel's tiles take well: the tcgen05 kernel.  Two MMA tiles per warp halve what reads the keys twice (24.6
    // against 29.4 us for 16 f32 rows, dim 128; 177 against 210 for 32 bf16 rows, dim 64) but not with all 16 rows of
    // dim 128 in use (176 against 154 us for 28 bf16 rows); dim 256 has no registers for them and two tiles read the keys twice
    // (37 against 48 us for 16 f32 rows).
    p.tensor = bound > (dim == 128 && !p.two ? unit : 2 * unit);
    p.mt = bound > unit && dim <= 128 ? 2 : 1;
    p.rows = p.tensor ? (dim == 256 || f32 || bound <= 128 ? 128 : 256) : (int)unit * p.mt;
    p.block = p.tensor && dim != 256 ? 128 : 64;
    const unsigned long long by_seq = (unsigned long long)n_seqs * ((bound + p.rows - 1) / p.rows), by_row = (unsigned long long)M * group / p.rows + n_seqs;
    p.tiles = (long long)(by_seq <= by_row ? by_seq : by_row);
    p.per_seq = by_seq <= by_row ? (int)((bound + p.rows - 1) / p.rows) : 0;
    size_t span = max_len;                                   // keys a tile can see at most
    if (window && window + p.rows < span) span = window + p.rows;
    const double blocks = (double)(span / p.block + 2), ctas = (double)p.tiles * (double)kv_heads;
    // Times in key blocks (about 1.5 us).  A CTA costs its start and end, hidden by its neighbour where two share an SM, and its blocks.
    // Lengths are bounds: of many sequences most are shorter, about half as long on average.  CTAs are handed to `slots` places as
    // they come free, so that the last ends about half a CTA after the work would on average.  Splits that do not join as a cluster
    // cost a launch, and the bytes of their sums.  (One 131 000-key pair of sequences: 135 us in 16 to 18 splits, 150 in 63; 64 ragged sequences of up to 8192
    // keys: 202 us in one split, 186 in 3 or 4, 214 in 12; 16 of up to 6000 with dim 256: 132, 43 in 4, 37 in 6, 50 in 16.  64 sequences
    // that all have 8192 keys: 340 us, 97 % of the copy rate, as they are planned here.)
    const bool pairs = dim != 256 && p.mt == 1 && !p.tensor;
    const double slots = (double)ctx->sm_count * (pairs ? 2 : 1), fixed = pairs ? 3.0 : 6.0, part = 0.5 + 0.5 / (double)n_seqs;
    const double sums = 0.25 + (double)M * (double)q_heads * (double)dim * 4.0 / 6.75e6;
    const int largest = p.tensor ? 1 : cluster_limit(ctx->device, pairs);
    double best = 0.0;
    int splits = 1;
    for (int n = 1; n <= 64 && n * 2 <= (int)blocks; n = n < 8 ? n + 1 : n + n / 4) {
        const double each = fixed + blocks / n, all = ctas * n, spread = part * all * each / slots + 0.5 * each;
        const bool cluster = !p.tensor && n <= largest && all <= slots;
        const double cost = (all <= slots || each > spread ? each : spread) + (n == 1 ? 0.0 : cluster ? 0.1 * n : 3.0 + sums * n);
        if (n == 1 || cost < best) { best = cost; splits = n; }
    }
    p.split_blocks = (int)((blocks + splits - 1) / splits);
    p.splits = (int)(((long long)blocks + p.split_blocks - 1) / p.split_blocks);
    const size_t rows = M * q_heads;
    p.cluster = !p.tensor && p.splits > 1 && p.splits <= largest && ctas * p.splits <= slots;
    p.workspace = p.splits > 1 && !p.cluster ? align256((size_t)p.splits * rows * sizeof(float2)) + (size_t)p.splits * rows * dim * sizeof(float) : 0;
    return p;
}

extern "C" int ojas_b200_attention_check(uint32_t cache_type, size_t page_size, size_t kv_heads, size_t dim, uint32_t act_type, size_t q_heads, const void *q,
                                         size_t q_stride, const void *out, size_t out_stride, float scale, int causal, long long window,
                                         const ojas_b200_seqs *seqs, size_t M, char *err, size_t errlen) {
    auto no = [&](int code, const char *why) { if (err && errlen) snprintf(err, errlen, "attention: %s", why); return code; };
    int rc = seqs_check(seqs, M, err, errlen);
    if (rc) return rc;
    rc = attn_shape_check(cache_type, page_size, kv_heads, dim, act_type, q_heads, M, seqs->max_rows, seqs->max_len, err, errlen);
    if (rc) return rc;
    if (!isfinite(scale * LOG2_E)) return no(OJAS_B200_E_ARG, "the scale, in powers of two, must be finite");
    if (window < 0 || window > 0x7fffffff) return no(OJAS_B200_E_ARG, "the window must be 0 (none) or a number of keys");
    if (window && !causal) return no(OJAS_B200_E_UNSUPPORTED, "a window needs causal rows");
    if ((q_stride && q_stride < q_heads * dim) || (out_stride && out_stride < q_heads * dim)) return no(OJAS_B200_E_ARG, "a row stride is smaller than a row");
    if (q_stride > (1ull << 40) || out_stride > (1ull << 40)) return no(OJAS_B200_E_LIMIT, "a stride is too large");
    if (q_stride % 4 || out_stride % 4) return no(OJAS_B200_E_ARG, "strides must be multiples of 4 elements");
    if (M && seqs->n_seqs) {
        if (!q || !out) return no(OJAS_B200_E_ARG, "null pointer");
        if ((uintptr_t)q % 16 || (uintptr_t)out % 16) return no(OJAS_B200_E_ARG, "q and out must start on 16 bytes");
    }
    return 0;
}

extern "C" size_t ojas_b200_attention_workspace_bytes(ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const ojas_b200_seqs *seqs, uint32_t act_type, size_t M, size_t q_heads,
                                                      long long window) {
    if (!ctx || !kv || !seqs || window < 0 || M == 0 || seqs->n_seqs == 0) return 0;
    if (attn_shape_check(kv->type, kv->page_size, kv->heads, kv->dim, act_type, q_heads, M, seqs->max_rows, seqs->max_len, nullptr, 0)) return 0;
    return attn_plan(ctx, seqs->n_seqs, M, seqs->max_rows, seqs->max_len, q_heads, kv->heads, kv->dim, (size_t)window, act_type == OJAS_B200_F32).workspace;
}

template <int D, bool BF, bool TWO, int MT>
static cudaError_t launch_rows(const ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p) {
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = smem_once(ready, ctx->device, attn_rows_kernel<D, BF, TWO, MT>, ar_smem(D), p.cluster && p.splits > 8);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.tiles, (unsigned)kv->heads, (unsigned)p.splits);
    cfg.blockDim = dim3(AR_THREADS);
    cfg.dynamicSmemBytes = ar_smem(D);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (ctx->pdl) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (p.cluster) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = 1;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = (unsigned)p.splits;
    }
    return cudaLaunchKernelEx(&cfg, attn_rows_kernel<D, BF, TWO, MT>, kv->map_k, kv->map_v, a, kv->box_rows);
}
template <int D, bool BF, bool TWO>
static cudaError_t launch_rows_form(const ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p) {
    return p.mt == 2 ? launch_rows<D, BF, TWO, D == 256 ? 1 : 2>(ctx, kv, a, p) : launch_rows<D, BF, TWO, 1>(ctx, kv, a, p);
}
template <bool BF>
static cudaError_t launch_rows_dim(const ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p) {
    if (kv->dim == 64) return p.two ? launch_rows_form<64, BF, true>(ctx, kv, a, p) : launch_rows_form<64, BF, false>(ctx, kv, a, p);
    if (kv->dim == 128) return p.two ? launch_rows_form<128, BF, true>(ctx, kv, a, p) : launch_rows_form<128, BF, false>(ctx, kv, a, p);
    return p.two ? launch_rows_form<256, BF, true>(ctx, kv, a, p) : launch_rows_form<256, BF, false>(ctx, kv, a, p);
}

extern "C" int ojas_b200_attention(ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const ojas_b200_seqs *seqs, uint32_t act_type, const void *q, size_t q_stride,
                                   size_t q_heads, float scale, int causal, long long window, void *out, size_t out_stride, size_t M, void *workspace,
                                   size_t workspace_bytes) {
    if (!ctx) return OJAS_B200_E_ARG;
    if (!kv) return ojas_fail(ctx, OJAS_B200_E_ARG, "attention: null cache");
    if (kv->device != ctx->device) return ojas_fail(ctx, OJAS_B200_E_ARG, "attention: the cache lives on device %d, the context on %d", kv->device, ctx->device);
    char why[256];
    const int rc = ojas_b200_attention_check(kv->type, kv->page_size, kv->heads, kv->dim, act_type, q_heads, q, q_stride, out, out_stride, scale, causal, window, seqs, M, why, sizeof why);
    if (rc) return ojas_fail(ctx, rc, "%s", why);
    if (M == 0 || seqs->n_seqs == 0) return 0;
    const AttnPlan p = attn_plan(ctx, seqs->n_seqs, M, seqs->max_rows, seqs->max_len, q_heads, kv->heads, kv->dim, (size_t)window, act_type == OJAS_B200_F32);
    if (p.workspace) {
        if (!workspace || workspace_bytes < p.workspace) return ojas_fail(ctx, OJAS_B200_E_ARG, "attention: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, p.workspace);
        if ((uintptr_t)workspace % 256) return ojas_fail(ctx, OJAS_B200_E_ARG, "attention: the workspace must start on 256 bytes");
    }
    if (p.tiles * (long long)kv->heads > 0x7fffffffll || p.splits > 65535) return ojas_fail(ctx, OJAS_B200_E_LIMIT, "attention: too many row tiles");
    AttnArgs a{};
    a.q = q; a.out = out;
    a.q_stride = (long long)(q_stride ? q_stride : q_heads * kv->dim);
    a.out_stride = (long long)(out_stride ? out_stride : q_heads * kv->dim);
    a.batch = {seqs->cu, seqs->len, seqs->table, (int)seqs->n_seqs, (int)seqs->table_stride, (long long)M, (int)kv->pages, (int)kv->page_size, (int)seqs->max_rows, ctx->dev_status};
    a.act_type = act_type; a.q_heads = (int)q_heads; a.group = (int)(q_heads / kv->heads);
    a.splits = p.splits; a.split_blocks = p.split_blocks; a.per_seq = p.per_seq;
    a.window = (int)window; a.causal = causal != 0;
    a.scale_log2 = scale * LOG2_E;
    if (p.workspace) {
        a.part_ml = static_cast<float2 *>(workspace);
        a.part_o = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + align256((size_t)p.splits * M * q_heads * sizeof(float2)));
    }
    DeviceGuard guard(ctx->device);
    cudaError_t e;
    if (p.tensor) {
        const int trc = attn_tc_launch(ctx, kv, a, p);
        if (trc) return trc;
    } else {
        e = kv->type == OJAS_B200_BF16 ? launch_rows_dim<true>(ctx, kv, a, p) : launch_rows_dim<false>(ctx, kv, a, p);
        if (e != cudaSuccess) return ojas_fail(ctx, OJAS_B200_E_CUDA, "launch attn_rows: %s", cudaGetErrorString(e));
        OJAS_LAUNCH_CHECK(ctx, "attn_rows");
    }
    if (p.splits > 1 && !p.cluster) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((M * q_heads + 7) / 8)); cfg.blockDim = dim3(256); cfg.stream = ctx->stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = ctx->pdl ? 1 : 0;
        e = kv->dim == 64 ? cudaLaunchKernelEx(&cfg, attn_join_kernel<64>, a)
                          : kv->dim == 128 ? cudaLaunchKernelEx(&cfg, attn_join_kernel<128>, a) : cudaLaunchKernelEx(&cfg, attn_join_kernel<256>, a);
        if (e != cudaSuccess) return ojas_fail(ctx, OJAS_B200_E_CUDA, "launch attn_join: %s", cudaGetErrorString(e));
        OJAS_LAUNCH_CHECK(ctx, "attn_join");
    }
    return 0;
}
