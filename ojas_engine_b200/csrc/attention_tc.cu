// Attention for many rows per key head (prompts, chunks of prompts, many query heads to a key head) on the 5th-generation
// tensor cores: S = Q K^T and O += P V as tcgen05.mma with f32 accumulators in TMEM, tensor-bound (4 dim flops a pair).
//
// A CTA takes NQ tiles of 128 rows (rows = token * group + head in group, so a short chunk still fills tiles) of one key head and a
// range of key blocks.  One warp copies K and V blocks from the pages into a ring (tensor copies, 128-byte swizzle), one thread
// issues the MMAs, and four warps per tile (NQ 1: eight) do the softmax: thread = row = TMEM lane (NQ 1: two threads to a row), its scores come out of TMEM into
// registers, the running maximum and sum stay in registers, and the probabilities go back into TMEM, where the second product
// reads them as its A operand.  Q stays in shared memory, O in TMEM.
//   NQ = 2 (dim 64 and 128, 16-bit activations): while one tile's softmax runs the tensor cores work for the other tile.  (Blocks of
//          64 keys would leave TMEM for probabilities beside the scores and let the scores run ahead, but every group of MMAs with a
//          completion signal takes 300 cycles at least and N = 64 is bound by shared memory: 828 against 565 us for an 8192-token prompt.)
//   NQ = 1 (dim 256, whose O takes half of TMEM, f32 activations, and calls of at most 128 rows per key head): two score buffers,
//          whose columns the probabilities reuse; the next block's scores are formed while the softmax runs.
// The accumulator is rescaled only when a row's maximum has grown by more than AT_SLACK (in log2) since it was last fixed, or a
// block's probabilities would leave f16's range (rare after the first blocks): they are kept scaled by 2^AT_SHIFT, below
// f16's limit and above its smallest values.
//
// f32 activations enter as two 16-bit terms (TERMS = 2): Q = Qhi + Qlo against the same K, P = Phi + Plo against the same V, twice the
// MMAs; rows of q are scaled by a power of two so that both terms are in f16's range.  16-bit activations are exact as they
// are and P is rounded once (by 2^-11 at most for f16, 2^-8 for bf16, random over the keys): results of unit-normal values are off by
// 2.6e-4 and 2.3e-3 of their norm, 2.0e-4 and 1.7e-3 of it the rounding of the result itself.  Two terms of P for them too would
// take an 8192-token f16 prompt from 613 to 801 us, a window of 1024 over heads of 64 from 111 to 125, 35 drafted rows from 25.4 to 27.1.
//
// The tensor cores cut what they add to an accumulator: every instruction takes up to 2^-23 off |O|, always towards zero, and
// thousands of them over a long context took 1.2e-5 off an f32 result (12 000 keys).  With f32 activations O is therefore added,
// in rounded f32, to sums of its own every 512 keys: in TMEM, or for dim 256, which leaves no room there, in the row's place
// in memory.
#include "attention.cuh"

namespace {

constexpr float AT_SHIFT = 8.0f, AT_SLACK = 7.0f;
constexpr float AT_SUM_MOST = 49152.0f;                    // (a block of 128 scores at the maximum gives 128 * 2^AT_SHIFT = 32768)
constexpr int AT_ROWS = 128;
constexpr int AT_MAX_STAGES = 10;

template <int D, int TERMS, int TILES>
struct AtShape {
    static constexpr int NQ = TILES;                                   // row tiles of a CTA
    static_assert(NQ == 1 || (TERMS == 1 && D <= 128), "two tiles' accumulators and q");
    static constexpr int KEYS = D == 256 ? 64 : 128;                   // keys of a block
    static constexpr bool AHEAD = NQ == 1;                             // a block's scores are formed before the products of the one before
    static constexpr int STAGE = KEYS * D * 2;                         // one block of K or V
    static constexpr int Q_TERM = AT_ROWS * D * 2, Q_BYTES = NQ * TERMS * Q_TERM;
    static constexpr int SHARE = NQ == 1 ? 2 : 1;                      // threads that share a row: one tile alone needs eight warps to hide latencies
    static constexpr int SMALL = 512 + (SHARE == 2 ? 2 * AT_ROWS * 4 : 0);           // barriers, and what the two threads of a row tell each other
    static constexpr int STAGES_FIT = (232448 - 1024 - SMALL - Q_BYTES) / STAGE;
    static constexpr int STAGES = STAGES_FIT > AT_MAX_STAGES ? AT_MAX_STAGES : STAGES_FIT;
    static constexpr int SMEM = Q_BYTES + STAGES * STAGE + SMALL + 1024;
    static constexpr int COLS = KEYS / SHARE, OUT = D / SHARE;         // scores, and columns of O, of a softmax thread
    static constexpr int SOFT_WARPS = 4 * NQ * SHARE, THREADS = (SOFT_WARPS + (NQ == 2 ? 4 : 2)) * 32;   // (NQ 2: whole warpgroups, see the register split)
    // TMEM columns: scores (NQ 1: two buffers), whose columns the probabilities reuse; O; (TERMS 2, dim <= 128) the sums of earlier blocks.
    static constexpr int FLUSH = TERMS == 2 ? 512 / KEYS : 1 << 30;    // blocks after which O is added to the sums
    static __host__ __device__ constexpr int col_s(int u, int n) { return NQ == 2 ? u * 128 : (n & 1) * 128; }
    static __host__ __device__ constexpr int col_o(int u) { return 256 + u * 128; }
    static constexpr int COL_SUM = 384;
    static constexpr int CHUNK = Q_BYTES / (SOFT_WARPS * 32) < 256 ? Q_BYTES / (SOFT_WARPS * 32) : 256;   // bytes of a row that the epilogue stages at a time
    static_assert(SOFT_WARPS * 32 * CHUNK <= Q_BYTES, "the epilogue stages rows where Q was");
    static_assert(CHUNK >= 64 && OUT % 32 == 0, "a chunk is 16 or whole 32s of f32 columns, whole 32s of 16-bit ones");
    static_assert(STAGES >= 3, "a K and a V block in use and one on the way");
};

__device__ __forceinline__ void at_ld32(uint32_t taddr, float *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                   "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                   "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
                   "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void at_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void at_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                   "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void at_st32f(uint32_t taddr, const float *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
                   "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]),
                   "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]) : "memory");
}
__device__ __forceinline__ void at_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Bounded wait without a call (ptxas splits registers between the roles only in code without calls).  Whole warps or one thread.
__device__ __forceinline__ bool at_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, unsigned *status) {
    if (mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(bar, parity)) {
        if (*abort_flag) return false;
        if (clock64() - t0 > WAIT_CYCLES) {
            *abort_flag = 1;
            atomicOr(status, OJAS_ST_ATTN_WAIT);
            __threadfence_system();
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool at_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_flag, unsigned *status) {
    return __all_sync(0xffffffffu, at_wait(bar, parity, abort_flag, status));
}

// One lane of a converged warp, chosen by the hardware: the compiler then knows that one thread issues what follows.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

// Shared-memory operands: the upper word of the descriptor is the same for all of them (groups of eight rows 1024 bytes apart,
// version 1, 128-byte swizzle), the lower one holds the address and, for V, the distance of its 64-column slabs.
constexpr uint32_t AT_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t at_desc(uint32_t smem_addr, uint32_t slab) { return ((smem_addr & 0x3FFFFu) >> 4) | (slab >> 4) << 16; }
// D = A B (accumulate 0) or D += A B; A from shared memory, or from TMEM.  The issuing warp shares its scheduler with two softmax
// warps: what it does per instruction has to stay below the 64 cycles an instruction takes, so the operands are kept where the
// compiler sees that they are the same in all lanes.
__device__ __forceinline__ void at_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(AT_DESC_HI) : "memory");
}
__device__ __forceinline__ void at_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(AT_DESC_HI) : "memory");
}
// kind::f16: f32 accumulator, M = 128, N = n; `mn`: B is stored with N contiguous (the rows of V: dim).
__host__ __device__ constexpr uint32_t at_idesc(int n, bool bf, bool mn) {
    return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
}
// sums = sums * by + O (first time: sums = O) for this thread's part of its row; O may then be overwritten.
template <int D, int OUT>
__device__ __forceinline__ void add_to_sums(uint32_t o_col, uint32_t sum_col, float *sums, bool live, bool more, float by) {
#pragma unroll 1
    for (int c = 0; c < OUT; c += 32) {
        float o[32];
        at_ld32(o_col + c, o);
        if (D <= 128) {
            if (more) {
                float e[32];
                at_ld32(sum_col + c, e);
                at_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = fmaf(e[i], by, o[i]);
            }
            at_wait_ld();
            at_st32f(sum_col + c, o);
        } else {
            at_wait_ld();
            if (live) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float4 v = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    if (more) {
                        const float4 e = *reinterpret_cast<const float4 *>(sums + c + i);
                        v = make_float4(fmaf(e.x, by, v.x), fmaf(e.y, by, v.y), fmaf(e.z, by, v.z), fmaf(e.w, by, v.w));
                    }
                    *reinterpret_cast<float4 *>(sums + c + i) = v;
                }
            }
            __syncwarp();
        }
    }
}

// The lowest n bits (n below 0: none, above 32: all).
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// The barrier of the two warps that share 32 rows.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, 64, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"((uint32_t)v), "r"(id) : "memory");
    return r != 0;
}

// Two values as two terms each: v = hi + lo.
template <bool BF>
__device__ __forceinline__ void split_two(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = pack_half(a, b, BF);
    const float2 h = unpack_half(hi, BF);
    lo = pack_half(a - h.x, b - h.y, BF);
}

// This thread's row of q, or its half of it (nothing: zeros), into shared memory as K-major operand tiles, one per term: all its
// loads first.  Returns the row's factor: score -> q . k.  told: where the threads of a row exchange the row's largest value.
template <int D, bool BF, int TERMS, int SHARE>
__device__ __forceinline__ float load_q(const void *q, long long at, bool live, float sign, unsigned char *tile, int r, int half, float *told, int mine,
                                        int other, int pair_bar) {
    constexpr int N = D / SHARE;
    const int c0 = half * N;
    float factor = 1.0f;
    // elements c .. c + 7 of row r: slab c / 64, 16-byte piece (c % 64) / 8 swizzled by the row
    auto place = [&](int c) { return tile + (c >> 6) * (AT_ROWS * 128) + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4); };
    if (TERMS == 2) {
        const float *src = static_cast<const float *>(q) + at + c0;
        float4 v[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; i++) v[i] = live ? *reinterpret_cast<const float4 *>(src + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < N / 4; i++) top = fmaxf(top, fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
        if (SHARE == 2) {
            told[mine] = top;
            pair_sync(pair_bar);
            top = fmaxf(top, told[other]);
        }
        const uint32_t ex = __float_as_uint(top) & 0x7f800000u;            // as in the kernel for few rows
        const bool scalable = ex > 0x01000000u && ex < 0x7e000000u;
        const float by = scalable ? sign * __uint_as_float(0x7f000000u - ex) : sign;
        factor = scalable ? __uint_as_float(ex) : 1.0f;
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            uint4 hi, lo;
            split_two<BF>(v[2 * i].x * by, v[2 * i].y * by, hi.x, lo.x);
            split_two<BF>(v[2 * i].z * by, v[2 * i].w * by, hi.y, lo.y);
            split_two<BF>(v[2 * i + 1].x * by, v[2 * i + 1].y * by, hi.z, lo.z);
            split_two<BF>(v[2 * i + 1].z * by, v[2 * i + 1].w * by, hi.w, lo.w);
            *reinterpret_cast<uint4 *>(place(c0 + 8 * i)) = hi;
            *reinterpret_cast<uint4 *>(place(c0 + 8 * i) + AT_ROWS * D * 2) = lo;
        }
    } else {
        const uint16_t *src = static_cast<const uint16_t *>(q) + at + c0;  // rows start on 8 bytes
        uint2 v[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; i++) v[i] = live ? *reinterpret_cast<const uint2 *>(src + 4 * i) : make_uint2(0u, 0u);
        const uint32_t flip = sign < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < N / 8; i++)
            *reinterpret_cast<uint4 *>(place(c0 + 8 * i)) = make_uint4(v[2 * i].x ^ flip, v[2 * i].y ^ flip, v[2 * i + 1].x ^ flip, v[2 * i + 1].y ^ flip);
    }
    return factor;
}

template <int D, bool BF, int TERMS, int TILES>
__global__ void __launch_bounds__(AtShape<D, TERMS, TILES>::THREADS, 1) attn_tiles_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                                  const __grid_constant__ CUtensorMap map_v, const AttnArgs a, int box_rows) {
    using S = AtShape<D, TERMS, TILES>;
    constexpr int NQ = S::NQ, KEYS = S::KEYS, STAGES = S::STAGES, STAGE = S::STAGE;
    extern __shared__ unsigned char at_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)at_raw + 1023) & ~(uintptr_t)1023);
    unsigned char *ring = smem + S::Q_BYTES;
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + STAGES * STAGE);
    uint64_t *kv_full = bars, *kv_empty = kv_full + AT_MAX_STAGES, *s_full = kv_empty + AT_MAX_STAGES, *p_full = s_full + 2;
    uint64_t *o_done = p_full + 2, *q_full = o_done + 2, *raw = q_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(raw + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *told_stop = abort_flag + 2;                                                          // [warp]
    float *told = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(bars) + 512);            // [half][row]
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, split = blockIdx.z;
    const int kv_heads = a.q_heads / a.group, kvh = blockIdx.x % kv_heads;
    unsigned *status = a.batch.status;

    grid_launch_dependents();
    grid_dependency_wait();
    // long tiles first, of all heads: the last rows of a sequence see the most keys
    RowTile t;
    if (!find_tile(a, (gridDim.x - 1 - blockIdx.x) / kv_heads, NQ * AT_ROWS, lane, t)) return;
    const int rows = min(NQ * AT_ROWS, t.n_rows - t.row0);
    int lo, hi;
    key_range(a, t, t.row0, t.row0 + rows, lo, hi);
    const int all0 = lo / KEYS, all1 = hi > lo ? (hi + KEYS - 1) / KEYS : all0;
    const bool alone = a.splits == 1 || all1 - all0 <= a.split_blocks;
    if (alone && split > 0) return;
    const int blk0 = min(all1, all0 + split * a.split_blocks), blk1 = split == a.splits - 1 ? all1 : min(all1, blk0 + a.split_blocks);
    // each tile's own part of the blocks (a tile without rows: none)
    int first[NQ], last[NQ];
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        first[u] = last[u] = blk0;
        const int r0 = t.row0 + u * AT_ROWS, r1 = min(r0 + AT_ROWS, t.n_rows);
        if (r1 > r0) {
            int l, h;
            key_range(a, t, r0, r1, l, h);
            if (h > l) { first[u] = min(blk1, max(blk0, l / KEYS)); last[u] = max(first[u], min(blk1, (h + KEYS - 1) / KEYS)); }
        }
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(&kv_full[s], 1); mbar_init(&kv_empty[s], 1); }
        for (int u = 0; u < 2; u++) { mbar_init(&s_full[u], 1); mbar_init(&q_full[u], 4 * S::SHARE); }
        for (int u = 0; u < 2; u++) { mbar_init(&p_full[u], 4 * S::SHARE); mbar_init(&o_done[u], 1); }
        mbar_init(raw, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_v) : "memory");
    }
    if (warp == S::SOFT_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Register split (NQ 2): 384 threads are launched with 168 registers each; 2 * 224 + 56 = 3 * 168.
    if (warp < S::SOFT_WARPS) {
        if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---------------- softmax of tile u.  Where two threads share a row, each takes half of a block's keys (and of the output's
        // columns); both keep the same maximum, and agree on it and on giving up at the pair's barrier.
        const int u = NQ == 2 ? warp >> 2 : 0, half = S::SHARE == 2 ? warp >> 2 : 0, quarter = warp & 3, pair_bar = 1 + quarter;
        const int mine = half * AT_ROWS + quarter * 32 + lane, other = (1 - half) * AT_ROWS + quarter * 32 + lane;
        const int r0 = t.row0 + u * AT_ROWS, row = r0 + quarter * 32 + lane;
        const bool live = row < t.n_rows;
        unsigned char *q_tile = smem + u * TERMS * S::Q_TERM;
        const long long token = live ? t.token0 + row / a.group : 0;
        const int head = kvh * a.group + (live ? row % a.group : 0);
        float factor = load_q<D, BF, TERMS, S::SHARE>(a.q, token * a.q_stride + (long long)head * D, live, a.scale_log2 < 0.0f ? -1.0f : 1.0f, q_tile, quarter * 32 + lane, half, told, mine, other, pair_bar);
        factor = fminf(fmaxf(factor * fabsf(a.scale_log2), 1e-37f), 3e38f);  // a masked score (-inf) has to stay -inf when multiplied
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[u]);
        int see_lo = 0, see_hi = 0;
        if (live) row_range(a, t, row, see_lo, see_hi);
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t o_col = lane_base + S::col_o(u) + half * S::OUT;
        const long long slot = ((long long)split * a.batch.M + token) * a.q_heads + head;
        // dim 256: the sums of earlier blocks wait in the row's place in memory
        float *sums = TERMS == 2 && D == 256 ? (alone ? static_cast<float *>(a.out) + token * a.out_stride + (long long)head * D : a.part_o + slot * D) + half * S::OUT : nullptr;
        float m = live ? -INFINITY : 0.0f, l = 0.0f, m_sums = -INFINITY;   // (rows past the tile's last only keep out of the way)
        bool ok = true;
        auto o_wait = [&](int n) {                           // the product of block n is in O
            ok = ok && at_wait_warp(&o_done[u], (uint32_t)n & 1u, abort_flag, status);
            tc_fence_after();
            return ok;
        };
        for (int blk = first[u], n = 0; blk < last[u]; blk++, n++) {
            const uint32_t s_col = lane_base + S::col_s(u, n) + half * S::COLS, p_col = lane_base + S::col_s(u, n) + half * (S::COLS / 2);
            const int key0 = blk * KEYS + half * S::COLS;
            ok = ok && (NQ == 2 ? at_wait_warp(&s_full[u], (uint32_t)n & 1u, abort_flag, status) : at_wait_warp(&s_full[n & 1], (uint32_t)(n >> 1) & 1u, abort_flag, status));
            tc_fence_after();
            float x[S::COLS];
#pragma unroll
            for (int c = 0; c < S::COLS; c += 32) at_ld32(s_col + c, x + c);
            at_wait_ld();
            bool flushed = false;
            if (TERMS == 2 && n > 0 && n % S::FLUSH == 0) {
                o_wait(n - 1);
                add_to_sums<D, S::OUT>(o_col, lane_base + S::COL_SUM + half * S::OUT, sums, live, n > S::FLUSH, m_sums == m ? 1.0f : exp2_fast(m_sums - m));
                m_sums = m;
                flushed = true;
            }
            // Most blocks raise no row's maximum by much: their probabilities are formed against the maximum so far, without looking
            // for the block's own, and kept if their sum, and with it each of them, is in f16's range (NaN is not).
            const bool edge = live && (blk * KEYS < see_lo || (blk + 1) * KEYS > see_hi);
            if (__any_sync(0xffffffffu, edge)) {
#pragma unroll
                for (int c = 0; c < S::COLS; c += 32) {      // a bit for each of 32 keys that the row sees
                    const uint32_t seen = below(see_hi - key0 - c) & ~below(see_lo - key0 - c);
#pragma unroll
                    for (int i = 0; i < 32; i++) x[c + i] = seen >> i & 1u ? x[c + i] : -INFINITY;
                }
            }
            bool again = __any_sync(0xffffffffu, !ok || (live && m == -INFINITY));
            float more = 0.0f, slack = AT_SLACK;
            // The probabilities overwrite scores: not before the other thread of the row has read its own.
            if (S::SHARE == 2) pair_sync(pair_bar);
            if (!again) {
                const uint64_t by = pair(factor, factor), less = pair(AT_SHIFT - m, AT_SHIFT - m);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < S::COLS; c += 32) {
                    uint32_t p16[16], lo16[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float x0 = x[c + 2 * i], x1 = x[c + 2 * i + 1];
                        const uint64_t y = fma2(pair(x0, x1), by, less);
                        float p0, p1;
                        unpair(y, p0, p1);
                        p0 = exp2_fast(p0);
                        p1 = exp2_fast(p1);
                        sum[i & 1] = add2(sum[i & 1], pair(p0, p1));
                        if (TERMS == 2) split_two<BF>(p0, p1, p16[i], lo16[i]);
                        else p16[i] = pack_half(p0, p1, BF);
                    }
                    at_st16(p_col + c / 2, p16);
                    if (TERMS == 2) at_st16(p_col + KEYS / 2 + c / 2, lo16);
                }
                float s0, s1;
                unpair(add2(sum[0], sum[1]), s0, s1);
                more = s0 + s1;
                again = !__all_sync(0xffffffffu, more <= AT_SUM_MOST || !live);
                slack = 0.0f;
            }
            if (S::SHARE == 2) again = pair_any(pair_bar, again);
            if (again) {
                at_wait_st();                                // what a failed attempt stored is stored again
                float tops[4];                               // four chains: one would be COLS dependent steps
#pragma unroll
                for (int c = 0; c < 4; c++) tops[c] = fmaxf(x[c], x[c + 4]);
#pragma unroll
                for (int c = 8; c < S::COLS; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) tops[e] = max3(tops[e], x[c + e], x[c + e + 4]);
                float top = max3(fmaxf(tops[0], tops[1]), tops[2], tops[3]) * factor;
                if (S::SHARE == 2) {
                    told[mine] = top;
                    if (lane == 0) told_stop[warp] = !ok;
                    pair_sync(pair_bar);
                    top = fmaxf(top, told[other]);
                    ok = (told_stop[warp] | told_stop[warp ^ 4]) == 0;
                }
                if (!ok) break;
                const bool grow = top > m + slack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = grow ? top : m;
                    const float f = mn == m ? 1.0f : exp2_fast(m - mn);
                    m = mn;
                    l *= f;
                    if (n > 0 && !flushed) {
                        // (without AHEAD the product of the block before came ahead of these scores)
                        if (S::AHEAD) o_wait(n - 1);
#pragma unroll 1
                        for (int c = 0; c < S::OUT; c += 32) {
                            float o[32];
                            at_ld32(o_col + c, o);
                            at_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] *= f;
                            at_st32f(o_col + c, o);
                        }
                    }
                }
                const float off = m == -INFINITY ? 0.0f : m - AT_SHIFT;
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < S::COLS; c += 32) {
                    uint32_t hi16[16], lo16[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p0 = exp2_fast(fmaf(x[c + 2 * i], factor, -off)), p1 = exp2_fast(fmaf(x[c + 2 * i + 1], factor, -off));
                        part[i & 3] += p0 + p1;
                        if (TERMS == 2) split_two<BF>(p0, p1, hi16[i], lo16[i]);
                        else hi16[i] = pack_half(p0, p1, BF);
                    }
                    at_st16(p_col + c / 2, hi16);
                    if (TERMS == 2) at_st16(p_col + KEYS / 2 + c / 2, lo16);
                }
                more = (part[0] + part[1]) + (part[2] + part[3]);
            }
            l += more;
            at_wait_st();
            // With the scores a block ahead, passing these probabilities on only when the product before has ended keeps every waiter
            // within one phase of its barrier (a parity cannot tell a phase from the one two before).
            if (S::AHEAD && n > 0) o_wait(n - 1);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[u]);
        }
        // ---------------- the tile's rows: O / l to out, or O and (m, l) to the split's place
        const int blocks = last[u] - first[u];
        if (ok && blocks > 0) {
            if (S::AHEAD) o_wait(blocks - 1);
            else {
                ok = at_wait_warp(&o_done[u], 0u, abort_flag, status);
                tc_fence_after();
            }
        }
        if (S::SHARE == 2) {
            pair_sync(pair_bar);
            told[mine] = l;
            pair_sync(pair_bar);
            l += told[other];
        }
        if (ok) {
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f, sums_by = m_sums == m ? 1.0f : exp2_fast(m_sums - m);
            if (live && half == 0 && !alone) a.part_ml[slot] = make_float2(l != l && m == -INFINITY ? 0.0f : m, l);   // (nothing but NaN seen is not "no key")
            if (live && half == 0 && alone && a.part_ml) a.part_ml[token * a.q_heads + head] = make_float2(0.0f, -1.0f);
            if (alone || blk1 > blk0) {
                // Rows leave through the tile's part of Q's shared memory (its MMAs have ended), S::CHUNK bytes of each at a time, so
                // that a warp writes whole stretches of a row instead of one piece of 32 rows.
                const int es = alone && a.act_type != OJAS_B200_F32 ? 2 : 4, per = S::CHUNK / es;      // element size, columns of a chunk
                unsigned char *stage = smem + warp * (S::CHUNK * 32);
                unsigned char *to = alone ? static_cast<unsigned char *>(a.out) + (token * a.out_stride + (long long)head * D + half * S::OUT) * es
                                          : reinterpret_cast<unsigned char *>(a.part_o + slot * D + half * S::OUT);
                if (!live) to = nullptr;
                if (blocks == 0) asm volatile("barrier.cta.sync %0, %1;" ::"r"(9 + u), "n"(128 * S::SHARE) : "memory");   // no MMA has waited for all of Q here
                const float by = alone ? inv : 1.0f;
                const bool wide = !alone || a.out_stride * es % 16 == 0;
                constexpr int PIECES = S::CHUNK / 16, TURN = PIECES < 8 ? PIECES - 1 : 7;   // 16-byte pieces of a row's chunk; piece p of row r lies at p ^ (r & TURN)
#pragma unroll 1
                for (int c0 = 0; c0 < S::OUT; c0 += per) {
#pragma unroll 1
                    for (int c = c0 & ~31; c < c0 + per; c += 32) {                    // (16 f32 columns: the half of 32 that the chunk holds)
                        float o[32];
                        if (blocks > 0) {
                            at_ld32(o_col + c, o);
                            if (TERMS == 2 && blocks > S::FLUSH) {
                                float e[32];
                                if (D <= 128) at_ld32(lane_base + S::COL_SUM + half * S::OUT + c, e);
                                at_wait_ld();
                                if (D > 128) {
#pragma unroll
                                    for (int i = 0; i < 32; i++) e[i] = live ? sums[c + i] : 0.0f;
                                }
#pragma unroll
                                for (int i = 0; i < 32; i++) o[i] = fmaf(e[i], sums_by, o[i]);
                            }
                            at_wait_ld();
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = 0.0f;
                        }
                        unsigned char *row_at = stage + lane * S::CHUNK;
                        const int p0 = (c - c0) * es / 16;
                        if (es == 4) {
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                if (S::CHUNK >= 128 || (unsigned)(p0 + i) < (unsigned)PIECES)
                                    *reinterpret_cast<float4 *>(row_at + (((p0 + i) ^ (lane & TURN)) << 4)) = make_float4(o[4 * i] * by, o[4 * i + 1] * by, o[4 * i + 2] * by, o[4 * i + 3] * by);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                *reinterpret_cast<uint4 *>(row_at + (((p0 + i) ^ (lane & TURN)) << 4)) =
                                    make_uint4(pack_half(o[8 * i] * by, o[8 * i + 1] * by, BF), pack_half(o[8 * i + 2] * by, o[8 * i + 3] * by, BF),
                                               pack_half(o[8 * i + 4] * by, o[8 * i + 5] * by, BF), pack_half(o[8 * i + 6] * by, o[8 * i + 7] * by, BF));
                        }
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int i = 0; i < PIECES; i++) {
                        const int r = (i * 32 + lane) / PIECES, p = lane % PIECES;
                        unsigned char *row_to = reinterpret_cast<unsigned char *>(__shfl_sync(0xffffffffu, (unsigned long long)to, r));
                        const uint4 v = *reinterpret_cast<const uint4 *>(stage + r * S::CHUNK + ((p ^ (r & TURN)) << 4));
                        if (row_to) {
                            uint4 *dst = reinterpret_cast<uint4 *>(row_to + c0 * es + p * 16);
                            if (wide) *dst = v;
                            else {                           // 16-bit rows that start on 8 bytes
                                reinterpret_cast<uint2 *>(dst)[0] = make_uint2(v.x, v.y);
                                reinterpret_cast<uint2 *>(dst)[1] = make_uint2(v.z, v.w);
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else {
    if (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == S::SOFT_WARPS) {
        // ---------------- MMA issue: the warp waits together, one elected lane issues (one warp for both tiles: with one each their
        // MMAs mix, and both tiles wait longer for theirs).  Ring order: see the loader.
        constexpr uint32_t ID_S = at_idesc(KEYS, BF, false), ID_O = at_idesc(D, BF, true);
        bool ok = true;
        const int b0 = __shfl_sync(0xffffffffu, blk0, 0), b1 = __shfl_sync(0xffffffffu, blk1, 0);
        int from[NQ], to[NQ];
#pragma unroll
        for (int u = 0; u < NQ; u++) { from[u] = __shfl_sync(0xffffffffu, first[u], 0); to[u] = __shfl_sync(0xffffffffu, last[u], 0); }
        int s = 0;
        uint32_t phase = 0;
        const uint32_t ring_at = __shfl_sync(0xffffffffu, smem_u32(ring), 0), q_at = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        auto next = [&]() { if (++s == STAGES) { s = 0; phase ^= 1u; } };
        auto wait = [&](uint64_t *bar, uint32_t parity) { ok = ok && at_wait_warp(bar, parity, abort_flag, status); };
        auto scores = [&](int u, int n, int stage) {
            const uint32_t kd = at_desc(ring_at + stage * STAGE, 16);
#pragma unroll
            for (int term = 0; term < TERMS; term++) {     // the low term first, while the sums are small
                const uint32_t qd = at_desc(q_at + (u * TERMS + TERMS - 1 - term) * S::Q_TERM, 16);
#pragma unroll
                for (int k = 0; k < D / 16; k++)           // 16 of dim: 32 bytes of a row, four per slab
                    at_mma_ss(tm + S::col_s(u, n), qd + (k >> 2) * (AT_ROWS * 128 / 16) + (k & 3) * 2, kd + (k >> 2) * (KEYS * 128 / 16) + (k & 3) * 2, ID_S,
                              term + k > 0);
            }
            umma_commit(&s_full[NQ == 2 ? u : n & 1]);
        };
        auto values = [&](int u, int n, int stage, bool last_block) {
            const uint32_t vd = at_desc(ring_at + stage * STAGE, KEYS * 128);
#pragma unroll
            for (int term = 0; term < TERMS; term++)
#pragma unroll
                for (int k = 0; k < KEYS / 16; k++)        // 16 keys: 8 columns of packed P, 2048 bytes of V
                    at_mma_ts(tm + S::col_o(u), tm + S::col_s(u, n) + term * (KEYS / 2) + k * 8, vd + k * (2048 / 16), ID_O, n % S::FLUSH != 0 || term + k > 0);
            if (S::AHEAD || last_block) umma_commit(&o_done[u]);
        };
        for (int u = 0; u < NQ; u++)
            if (to[u] > from[u]) wait(&q_full[u], 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        int n_s[NQ] = {}, n_o[NQ] = {};                      // blocks of a tile whose scores, whose products have been issued
        for (int i = b0; ok && i <= b1; i++) {
            if (S::AHEAD) {
                // (K0) (K1 V0) (K2 V1) ... (Vlast): block i's scores, then the products of block i - 1
                if (i < b1) {
                    wait(&kv_full[s], phase);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        scores(0, n_s[0], s);
                        umma_commit(&kv_empty[s]);
                    }
                    __syncwarp();
                    n_s[0]++;
                    next();
                }
                if (i > b0) {
                    wait(&kv_full[s], phase);
                    wait(&p_full[0], (uint32_t)n_o[0] & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        values(0, n_o[0], s, i == to[0]);
                        umma_commit(&kv_empty[s]);
                    }
                    __syncwarp();
                    n_o[0]++;
                    next();
                }
            } else {
                // (K0) (V0 K1) (V1 K2) ... (Vlast): a tile's products, then its next scores over the probabilities they read
                const int v_stage = s;
                if (i > b0) { wait(&kv_full[s], phase); next(); }
                const int k_stage = s;
                const uint32_t k_phase = phase;
                if (i < b1) next();
#pragma unroll
                for (int u = 0; u < NQ; u++) {
                    const bool has_o = i - 1 >= from[u] && i - 1 < to[u], has_s = i >= from[u] && i < to[u];
                    if (has_o) wait(&p_full[u], (uint32_t)n_o[u] & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        if (has_o) values(u, n_o[u], v_stage, i == to[u]);
                        if (u == NQ - 1 && i > b0) umma_commit(&kv_empty[v_stage]);
                    }
                    __syncwarp();
                    n_o[u] += has_o;
                    if (u == 0 && i < b1) wait(&kv_full[k_stage], k_phase);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        if (has_s) scores(u, n_s[u], k_stage);
                        if (u == NQ - 1 && i < b1) umma_commit(&kv_empty[k_stage]);
                    }
                    __syncwarp();
                    n_s[u] += has_s;
                }
            }
        }
    } else if (warp == S::SOFT_WARPS + 1) {
        // ---------------- loader: lane = one box (64 values x box_rows tokens); K0 K1 V0 K2 V1 ... Vlast, or (not AHEAD) K0 V0 K1 V1 ...
        const int per_slab = KEYS / box_rows, part = lane % per_slab, slab = lane / per_slab;
        const bool has_box = slab < D / 64;
        const int *table = a.batch.table + (long long)t.seq * a.batch.table_stride;
        const int page_size = a.batch.page_size, step_entry = KEYS / page_size, step_slot = KEYS - step_entry * page_size;
        int s = 0;
        uint32_t phase = 1, raw_phase = 0;
        bool ok = true;
        // this lane's box of block blk: the page (looked up a block ahead of its use, -1: not needed) and the token in it
        int key = blk0 * KEYS + part * box_rows, entry = key / page_size, slot = key - entry * page_size;
        auto look_up = [&]() { return has_box && key < hi && key + box_rows > lo ? __ldg(table + entry) : -1; };
        auto advance = [&]() {
            key += KEYS;
            entry += step_entry;
            slot += step_slot;
            if (slot >= page_size) { slot -= page_size; entry++; }
        };
        auto copy = [&](const CUtensorMap *map, bool is_v, int blk, bool want, int page, int at) {
            ok = ok && at_wait_warp(&kv_empty[s], phase, abort_flag, status);
            if (!ok) return;
            unsigned char *to = ring + s * STAGE;
            const int copies = __popc(__ballot_sync(0xffffffffu, want));
            // the values of keys that are not read must be zeros (0 * NaN is NaN): such a block lands on a barrier of the loader's own
            // and is passed on after they are
            const bool edge = is_v && (blk * KEYS < lo || (blk + 1) * KEYS > hi);
            uint64_t *bar = edge ? raw : &kv_full[s];
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(copies * box_rows * 128));
            __syncwarp();
            if (want) tma_load_4d(to + slab * (KEYS * 128) + part * box_rows * 128, map, slab * 64, at, kvh, page, bar);
            if (edge) {
                ok = at_wait_warp(raw, raw_phase, abort_flag, status);
                raw_phase ^= 1u;
                for (int e = lane; e < KEYS * (D / 8); e += 32) {          // 16-byte pieces; a row's pieces may be zeroed in any order
                    const int r = e / (D / 8), c = e % (D / 8);
                    if (blk * KEYS + r < lo || blk * KEYS + r >= hi) *reinterpret_cast<uint4 *>(to + (c >> 3) * (KEYS * 128) + r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&kv_full[s]);
            }
            if (++s == STAGES) { s = 0; phase ^= 1u; }
        };
        int next_page = blk0 < blk1 ? look_up() : -1, v_page = 0, v_slot = 0;
        bool v_want = false;
        for (int blk = blk0; blk < blk1 && ok; blk++) {
            const bool want = has_box && key < hi && key + box_rows > lo;
            int page = next_page;
            const int at = slot;
            if (want && (page < 0 || page >= a.batch.pages)) { atomicOr(status, OJAS_ST_BATCH); page = a.batch.pages; }   // reads as zeros
            advance();
            if (blk + 1 < blk1) next_page = look_up();
            copy(&map_k, false, blk, want, page, at);
            if (!S::AHEAD) copy(&map_v, true, blk, want, page, at);
            else if (blk > blk0) copy(&map_v, true, blk - 1, v_want, v_page, v_slot);
            v_want = want; v_page = page; v_slot = at;
        }
        if (S::AHEAD && blk1 > blk0) copy(&map_v, true, blk1 - 1, v_want, v_page, v_slot);
    }
    }

    // ---------------- teardown: every role arrives here, also after an abort (copies and MMAs in flight then get a bounded time)
    if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == S::SOFT_WARPS) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D, bool BF, int TERMS, int TILES>
cudaError_t launch_tiles(const ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p) {
    using S = AtShape<D, TERMS, TILES>;
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = smem_once(ready, ctx->device, attn_tiles_kernel<D, BF, TERMS, TILES>, S::SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.tiles * (long long)kv->heads), 1, (unsigned)p.splits);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, attn_tiles_kernel<D, BF, TERMS, TILES>, kv->map_k, kv->map_v, a, kv->box_rows);
}
template <bool BF, int TERMS>
cudaError_t launch_tiles_dim(const ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p) {
    constexpr int TWO = TERMS == 1 ? 2 : 1;
    if (kv->dim == 64) return p.rows == 256 ? launch_tiles<64, BF, TERMS, TWO>(ctx, kv, a, p) : launch_tiles<64, BF, TERMS, 1>(ctx, kv, a, p);
    if (kv->dim == 128) return p.rows == 256 ? launch_tiles<128, BF, TERMS, TWO>(ctx, kv, a, p) : launch_tiles<128, BF, TERMS, 1>(ctx, kv, a, p);
    return launch_tiles<256, BF, TERMS, 1>(ctx, kv, a, p);
}

}  // namespace

int attn_tc_launch(ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const AttnArgs &a, const AttnPlan &p) {
    const bool bf = kv->type == OJAS_B200_BF16, two = a.act_type == OJAS_B200_F32;
    const cudaError_t e = bf ? (two ? launch_tiles_dim<true, 2>(ctx, kv, a, p) : launch_tiles_dim<true, 1>(ctx, kv, a, p))
                             : (two ? launch_tiles_dim<false, 2>(ctx, kv, a, p) : launch_tiles_dim<false, 1>(ctx, kv, a, p));
    if (e != cudaSuccess) return ojas_fail(ctx, OJAS_B200_E_CUDA, "launch attn_tiles: %s", cudaGetErrorString(e));
    OJAS_LAUNCH_CHECK(ctx, "attn_tiles");
    return 0;
}
