// The rotation itself, shared by rope.cu and kv.cu: the angle of a pair, and what one thread does to one unit of a head.
#pragma once
#include <new>

#include "attn.cuh"

// cos and sin of pos * turns[i] turns, times the magnitude.  The product modulo 2^64 read as a signed fraction is the angle in
// (-1/2, 1/2] turns; the position may be negative (two's complement).
__device__ __forceinline__ float2 rope_angle(int pos, uint64_t turns, float magnitude) {
    const int64_t frac = (int64_t)((uint64_t)(int64_t)pos * turns);
    const float half_turns = (float)(int)(frac >> 32) * 4.656612873077393e-10f;   // 2^-31: units of pi
    float s, c;
    sincospif(half_turns, &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

// Units a head is cut into: VEC pairs each, then 2 VEC passing elements each.
__host__ __device__ inline int rope_units(int vec, int rot, int dim) { return rot / 2 / vec + (dim - rot + 2 * vec - 1) / (2 * vec); }
// Four pairs at a time need whole vectors in both halves of the rotated part and behind it.
static inline bool rope_vec_ok(int rot, int dim, bool) { return rot % 8 == 0 && (dim - rot) % 8 == 0; }
static inline bool rope_rows_aligned(const void *p, uint32_t type, long long stride) {
    return (uintptr_t)p % (4 * elem_bytes(type)) == 0 && stride % 4 == 0;
}

template <int VEC>
struct RopeUnit {
    int a, b, f;         // element offsets of the unit's two parts, index of its first frequency (-1: passes through, -2: nothing)
    bool inter;
    __device__ RopeUnit(int u, int rot, int dim, bool interleaved) : inter(interleaved) {
        const int turning = rot / 2 / VEC;
        if (u < turning) {
            f = u * VEC;
            a = interleaved ? 2 * u * VEC : u * VEC;
            b = interleaved ? a + VEC : a + rot / 2;
        } else {
            a = rot + (u - turning) * 2 * VEC;
            b = a + VEC;
            f = a < dim ? -1 : -2;
        }
    }
    // One head: x at element xo -> y at element yo.  x and y may be the same row: a thread reads all it writes first.
    __device__ __forceinline__ void apply(const void *x, uint32_t xt, long long xo, void *y, uint32_t yt, long long yo, const float2 *cs) const {
        if (f == -2) return;
        if (VEC == 4) {
            const float4 p = load_elem4(x, xt, xo + a), q = load_elem4(x, xt, xo + b);
            if (f < 0) {
                store_elem4(y, yt, yo + a, p);
                store_elem4(y, yt, yo + b, q);
                return;
            }
            const float4 *c4 = reinterpret_cast<const float4 *>(cs + f);
            const float4 c01 = c4[0], c23 = c4[1];             // (cos, sin) of two frequencies each
            float4 u, v;
            if (inter) {                                        // p = pairs 0, 1; q = pairs 2, 3
                u = make_float4(p.x * c01.x - p.y * c01.y, p.y * c01.x + p.x * c01.y, p.z * c01.z - p.w * c01.w, p.w * c01.z + p.z * c01.w);
                v = make_float4(q.x * c23.x - q.y * c23.y, q.y * c23.x + q.x * c23.y, q.z * c23.z - q.w * c23.w, q.w * c23.z + q.z * c23.w);
            } else {                                            // p = first members, q = second members
                u = make_float4(p.x * c01.x - q.x * c01.y, p.y * c01.z - q.y * c01.w, p.z * c23.x - q.z * c23.y, p.w * c23.z - q.w * c23.w);
                v = make_float4(q.x * c01.x + p.x * c01.y, q.y * c01.z + p.y * c01.w, q.z * c23.x + p.z * c23.y, q.w * c23.z + p.w * c23.w);
            }
            store_elem4(y, yt, yo + a, u);
            store_elem4(y, yt, yo + b, v);
        } else {
            const float p = load_elem(x, xt, xo + a), q = load_elem(x, xt, xo + b);
            float u = p, v = q;
            if (f >= 0) {
                const float2 c = cs[f];
                u = p * c.x - q * c.y;
                v = q * c.x + p * c.y;
            }
            store_elem(y, yt, yo + a, u);
            store_elem(y, yt, yo + b, v);
        }
    }
};
