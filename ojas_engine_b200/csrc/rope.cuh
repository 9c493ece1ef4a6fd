// The rotation itself, shared by rope.cu and kv.cu: the angle of a pair, and what one thread does to one unit of a head.
#pragma once
#include <new>

#include "attn.cuh"

// cos and sin of pos * turns[i] turns, times the magnitude.  The product modulo 2^64 read as a signed fraction is the angle in
// [-1/2, 1/2) turns; the position may be negative (two's complement).  An f32 holds the fraction's top 24 bits; the next 32, at most
// 3.7e-7 radians, turn sine and cosine to first order (the second is below 1e-13).  (Rounded to an f32 alone, the angle is off by up to 9.4e-8.)
__device__ __forceinline__ float2 rope_angle(int pos, uint64_t turns, float magnitude) {
    const uint64_t frac = (uint64_t)(int64_t)pos * turns;
    const int top = (int)(uint32_t)(frac >> 32) & ~0xff;
    const float rest = (float)(uint32_t)(frac >> 8) * 8.7196693e-17f;             // pi 2^-55: radians
    float s, c;
    sincospif((float)top * 4.656612873077393e-10f, &s, &c);                       // 2^-31: units of pi
    return make_float2(fmaf(-s, rest, c) * magnitude, fmaf(c, rest, s) * magnitude);
}

// Units a head is cut into: VEC pairs each, then 2 VEC passing elements each.
__host__ __device__ inline int rope_units(int vec, int rot, int dim) { return rot / 2 / vec + (dim - rot + 2 * vec - 1) / (2 * vec); }
// Four pairs at a time need whole vectors in both halves of the rotated part and behind it.
static inline bool rope_vec_ok(int rot, int dim) { return rot % 8 == 0 && (dim - rot) % 8 == 0; }
static inline bool rope_rows_aligned(const void *p, uint32_t type, long long stride) {
    return (uintptr_t)p % (4 * elem_bytes(type)) == 0 && stride % 4 == 0;
}

template <int VEC>
struct RopeUnit {
    // Element offsets of the unit's two parts, each VEC neighbouring elements so that a warp's accesses are whole stretches of a row;
    // the first frequencies of the pairs they belong to (f -1: passes through, -2: nothing).
    int a, b, f, f2;
    bool inter;
    __device__ RopeUnit(int u, int rot, int dim, bool interleaved) : inter(interleaved) {
        const int turning = rot / 2 / VEC;
        if (u < turning) {
            f = f2 = u * VEC;                                  // half: part a holds the pairs' first members, part b the second
            a = u * VEC;
            b = a + rot / 2;
            if (interleaved && VEC == 4) {                      // two pairs in each part
                f = 2 * u;
                f2 = f + rot / 4;
            } else if (interleaved) {
                a = 2 * u;
                b = a + 1;
            }
        } else {
            const int pass = u - turning, step = VEC == 4 ? (dim - rot) / 2 : 1;
            a = rot + pass * (VEC == 4 ? 4 : 2);
            b = a + step;
            f = f2 = b < dim ? -1 : -2;
        }
    }
    // One head's unit: x at element xo -> y at element yo, read and written apart so that a thread can read several heads before it
    // writes the first (the compiler has to assume that y is x).
    struct Parts { float4 a, b; };
    __device__ __forceinline__ void fetch(const void *x, uint32_t xt, long long xo, Parts &p) const {
        if (f == -2) return;
        if (VEC == 4) {
            p.a = load_elem4(x, xt, xo + a);
            p.b = load_elem4(x, xt, xo + b);
        } else {
            p.a.x = load_elem(x, xt, xo + a);
            p.b.x = load_elem(x, xt, xo + b);
        }
    }
    // angles: (cos, sin) of two pairs each, so that their type asks for the alignment with which they are read.
    __device__ __forceinline__ void put(const Parts &in, void *y, uint32_t yt, long long yo, const float4 *angles) const {
        if (f == -2) return;
        const float4 p = in.a, q = in.b;
        if (VEC == 4) {
            if (f < 0) {
                store_elem4(y, yt, yo + a, p);
                store_elem4(y, yt, yo + b, q);
                return;
            }
            // (cos, sin) of two frequencies each: pairs 0, 1 and 2, 3 of the unit
            const float4 c01 = angles[f >> 1], c23 = angles[inter ? f2 >> 1 : (f >> 1) + 1];
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
            float u = p.x, v = q.x;
            if (f >= 0) {
                const float2 c = reinterpret_cast<const float2 *>(angles)[f];
                u = p.x * c.x - q.x * c.y;
                v = q.x * c.x + p.x * c.y;
            }
            store_elem(y, yt, yo + a, u);
            store_elem(y, yt, yo + b, v);
        }
    }
};

// A thread's heads first, first + step, ... below `heads` of one token, ROPE_BATCH of them in flight.  rope_fetch may come before the
// angles are known: what a CTA waits for longest are its first loads, and those do not depend on them.  (Two heads in flight: 24.8 and
// 49.0 us for the rotation and the append of a prompt's chunk; one 26.0 and 54.9, four 25.5 and 51.0, eight 29.2 and 63.8, which leave fewer CTAs per SM.)
constexpr int ROPE_BATCH = 2;
template <int VEC>
__device__ __forceinline__ void rope_fetch(const RopeUnit<VEC> &unit, int first, int step, int heads, int dim, const void *x, uint32_t xt, long long xo,
                                           typename RopeUnit<VEC>::Parts (&p)[ROPE_BATCH]) {
    if (xt == OJAS_B200_F32) {                                  // (a constant type lets the loads go out together)
#pragma unroll
        for (int j = 0; j < ROPE_BATCH; j++)
            if (first + j * step < heads) unit.fetch(x, OJAS_B200_F32, xo + (long long)(first + j * step) * dim, p[j]);
    } else {
#pragma unroll
        for (int j = 0; j < ROPE_BATCH; j++)
            if (first + j * step < heads) unit.fetch(x, xt, xo + (long long)(first + j * step) * dim, p[j]);
    }
}
template <int VEC>
__device__ __forceinline__ void rope_put(const RopeUnit<VEC> &unit, int first, int step, int heads, int dim, void *y, uint32_t yt, long long yo, const float4 *angles,
                                         const typename RopeUnit<VEC>::Parts (&p)[ROPE_BATCH]) {
#pragma unroll
    for (int j = 0; j < ROPE_BATCH; j++)
        if (first + j * step < heads) unit.put(p[j], y, yt, yo + (long long)(first + j * step) * dim, angles);
}
