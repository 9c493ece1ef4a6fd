// Declarations shared by the operators between a layer's projections: rotary positions (rope.cu), the paged cache and
// the append (kv.cu), and attention over it (attention.cu, attention_tc.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"

// Rotation of one pair per frequency.  turns[i] is the frequency in turns per position as a 64-bit binary fraction, so
// pos * turns[i] modulo 2^64 is the pair's angle modulo one turn, exactly, for every 32-bit position.
struct ojas_b200_rope {
    int device;
    uint32_t rot_dim;
    float magnitude;
    uint64_t *turns;          // device, rot_dim / 2
};

struct ojas_b200_kv {
    int device;
    uint32_t type;            // OJAS_B200_F16 or OJAS_B200_BF16
    void *k, *v;
    size_t pages, page_size, heads, dim;
    size_t page_stride, head_stride, token_stride;   // elements
    int box_rows;             // tokens one tensor copy takes: the largest power of two up to 64 that divides a page
    CUtensorMap map_k, map_v;
};

// The batch as a kernel sees it.
struct BatchArgs {
    const int *cu, *len, *table;
    int n_seqs, table_stride;          // entries per sequence in the page table
    long long M;                       // rows of the call
    int pages, page_size, max_rows;
    unsigned *status;
};

static inline size_t elem_bytes(uint32_t type) { return type == OJAS_B200_F32 ? 4 : 2; }
static inline bool elem_type(uint32_t type) { return type == OJAS_B200_F32 || type == OJAS_B200_F16 || type == OJAS_B200_BF16; }

// Makes the context's device current for the time of a call.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before == device) before = -1;
        else cudaSetDevice(device);
    }
    ~DeviceGuard() { if (before >= 0) cudaSetDevice(before); }
};

// Checks that need no device; a message in err on refusal (kv.cu).
int seqs_check(const ojas_b200_seqs *s, size_t M, char *err, size_t errlen);

#ifdef __CUDACC__
// ---------------------------------------------------------------------------- element types at run time
__device__ __forceinline__ float load_elem(const void *p, uint32_t type, long long i) {
    if (type == OJAS_B200_F32) return static_cast<const float *>(p)[i];
    if (type == OJAS_B200_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_elem(void *p, uint32_t type, long long i, float v) {
    if (type == OJAS_B200_F32) static_cast<float *>(p)[i] = v;
    else if (type == OJAS_B200_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ uint32_t pack_half(float a, float b, bool bf) {
    if (bf) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t u, bool bf) {
    if (bf) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
// Four neighbouring elements, element index a multiple of 4 from a 16-byte (f32) or 8-byte (16-bit) boundary.
__device__ __forceinline__ float4 load_elem4(const void *p, uint32_t type, long long i) {
    if (type == OJAS_B200_F32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
    const float2 a = unpack_half(u.x, type == OJAS_B200_BF16), b = unpack_half(u.y, type == OJAS_B200_BF16);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store_elem4(void *p, uint32_t type, long long i, const float4 &v) {
    if (type == OJAS_B200_F32) *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = v;
    else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i) = make_uint2(pack_half(v.x, v.y, type == OJAS_B200_BF16), pack_half(v.z, v.w, type == OJAS_B200_BF16));
}

// ---------------------------------------------------------------------------- which sequence a row belongs to
// Rows [start, end) of a sequence lie in a call of M rows.
__device__ __forceinline__ bool seq_in_call(int start, int end, long long M) { return start >= 0 && end >= start && end <= M; }
// One warp, all lanes together: the sequence b with cu[b] <= row < cu[b + 1], or -1.  Each step narrows the range by 32.
// Out-of-order offsets give some sequence or -1, never an index outside the batch.
__device__ __forceinline__ int find_seq(const int *cu, int n_seqs, long long row, int lane) {
    int lo = 0, n = n_seqs;                       // the answer is in [lo, lo + n) if there is one
    while (n > 0) {
        const int step = (n + 31) >> 5;
        const int end = min((lane + 1) * step, n);
        const bool past = (long long)__ldg(cu + lo + end) <= row && lane * step < n;   // the lane's part ends before the row
        const int parts = __popc(__ballot_sync(0xffffffffu, past));
        lo += min(parts * step, n);
        if (parts * step >= n) return -1;         // behind the last sequence (or the end of a disordered range)
        n = min(step, n_seqs - lo);
        if (step == 1) break;
    }
    return lo < n_seqs && (long long)__ldg(cu + lo) <= row && (long long)__ldg(cu + lo + 1) > row ? lo : -1;
}
#endif
