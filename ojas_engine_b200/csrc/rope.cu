// Rotary positions: pair i of a head is turned by the angle pos * f_i,
//     (a, b) -> magnitude * (a cos - b sin, b cos + a sin),
// f_i = base^(-2i / rot_dim), scaled for contexts longer than the trained one.  Pairs are (x[i], x[i + rot_dim/2]) (half) or
// (x[2i], x[2i + 1]) (interleaved); elements from rot_dim on pass through.
//
// Angles: a 32-bit product pos * f_i is wrong by 0.06 radians at position 10^6.  The frequency is kept in turns as a 64-bit
// binary fraction instead: pos * turns wraps modulo 2^64, i.e. modulo one turn, without any rounding; rope_angle uses 56 bits of it.
// What is left is the frequency's own error times the position, so it is formed with 64-bit significands: steps of 2^-64 of f_i in pow,
// the scaling and the division by 2 pi, and half of 2^-64 turns, together below 2^-61 radians for f_i up to 1, 1e-9 radians at position
// 2^31.  (From a double's 53 bits it was 2.6e-7.)
#include <float.h>
#include <math.h>

#include "attn.cuh"
#include "rope.cuh"

static_assert(LDBL_MANT_DIG >= 64, "frequencies are formed with 64-bit significands");
constexpr long double TWO_PI = 6.283185307179586476925286766559005768L;

// The frequencies in radians per position (host).
static int rope_frequencies(size_t rot_dim, double base, const ojas_b200_rope_scaling *sc, const float *freq_factors, long double *f, char *err, size_t errlen) {
    auto no = [&](const char *why) { if (err && errlen) snprintf(err, errlen, "rope: %s", why); return OJAS_B200_E_ARG; };
    if (rot_dim < 2 || rot_dim % 2 != 0 || rot_dim > 1024) return no("rot_dim must be even, 2..1024");
    if (!(base > 1.0) || !isfinite(base)) return no("base must be a finite number above 1");
    const double factor = sc ? sc->factor : 1.0, fast = sc ? sc->beta_fast : 0.0, slow = sc ? sc->beta_slow : 0.0;
    if (!(factor > 0.0) || !isfinite(factor)) return no("factor must be positive");
    if (sc && !(sc->magnitude > 0.0f && isfinite(sc->magnitude))) return no("magnitude must be positive");
    if (sc && sc->orig_len && !(fast > slow && slow >= 0.0 && isfinite(fast))) return no("beta_fast must be above beta_slow, both finite and not negative");
    for (size_t i = 0; i < rot_dim / 2; i++) {
        f[i] = powl((long double)base, -2.0L * (long double)i / (long double)rot_dim);
        if (freq_factors) {
            if (!(freq_factors[i] > 0.0f) || !isfinite(freq_factors[i])) return no("frequency factors must be positive");
            f[i] /= (long double)freq_factors[i];
        }
        if (sc && sc->orig_len) {                 // by parts: pairs that turn often within the original context keep their frequency
            long double keep = ((long double)sc->orig_len * f[i] / TWO_PI - slow) / ((long double)fast - slow);
            keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
            f[i] = f[i] * keep + f[i] / factor * (1.0L - keep);
        } else {
            f[i] /= factor;
        }
        if (!isfinite((double)f[i])) return no("a frequency is not finite");
    }
    return 0;
}

extern "C" int ojas_b200_rope_frequencies(size_t rot_dim, double base, const ojas_b200_rope_scaling *scaling, const float *freq_factors,
                                          double *radians_out, char *err, size_t errlen) {
    if (!radians_out) return OJAS_B200_E_ARG;
    long double f[512];
    const int rc = rope_frequencies(rot_dim, base, scaling, freq_factors, f, err, errlen);
    for (size_t i = 0; !rc && i < rot_dim / 2; i++) radians_out[i] = (double)f[i];
    return rc;
}

extern "C" int ojas_b200_rope_create(ojas_b200_ctx *ctx, size_t rot_dim, double base, const ojas_b200_rope_scaling *scaling, const float *freq_factors,
                                     ojas_b200_rope **out) {
    if (!ctx || !out) return OJAS_B200_E_ARG;
    *out = nullptr;
    long double f[512];
    uint64_t turns[512];
    const int rc = rope_frequencies(rot_dim, base, scaling, freq_factors, f, ctx->err, sizeof ctx->err);
    if (rc) return rc;
    for (size_t i = 0; i < rot_dim / 2; i++) {
        const long double t = f[i] / TWO_PI, frac = t - floorl(t);           // below one turn per position in all real uses
        const long double steps = floorl(ldexpl(frac, 64) + 0.5L);
        turns[i] = steps < 18446744073709551616.0L ? (uint64_t)steps : 0u;   // (rounded up to a whole turn)
    }
    DeviceGuard guard(ctx->device);
    uint64_t *dev = nullptr;
    OJAS_CUDA(ctx, cudaMalloc((void **)&dev, rot_dim / 2 * sizeof(uint64_t)));
    const cudaError_t e = cudaMemcpy(dev, turns, rot_dim / 2 * sizeof(uint64_t), cudaMemcpyHostToDevice);
    if (e != cudaSuccess) {
        cudaFree(dev);
        return ojas_fail(ctx, OJAS_B200_E_CUDA, "rope_create: %s", cudaGetErrorString(e));
    }
    ojas_b200_rope *r = new (std::nothrow) ojas_b200_rope();
    if (!r) { cudaFree(dev); return ojas_fail(ctx, OJAS_B200_E_LIMIT, "rope_create: out of host memory"); }
    r->device = ctx->device; r->rot_dim = (uint32_t)rot_dim; r->turns = dev;
    r->magnitude = scaling ? scaling->magnitude : 1.0f;
    *out = r;
    return 0;
}

extern "C" void ojas_b200_rope_destroy(ojas_b200_rope *r) {
    if (!r) return;
    DeviceGuard guard(r->device);
    cudaFree(r->turns);
    delete r;
}

// ---------------------------------------------------------------------------- rows
struct RopeArgs {
    const void *x;
    void *y;
    const int *pos;
    const uint64_t *turns;
    float magnitude;
    long long x_stride, y_stride;      // elements between tokens
    uint32_t x_type, y_type;
    int heads, dim, rot;
    bool interleaved;
};

// One CTA per token: its first loads go out, then it forms the token's cosines and sines in shared memory; every thread owns one
// unit of a head (VEC pairs, or 2 VEC elements that pass through) and walks the heads.  HBM bound: x in, y out.
template <int VEC>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeArgs a) {
    extern __shared__ float4 rope_cs[];           // (cos, sin) of two pairs each
    grid_launch_dependents();
    grid_dependency_wait();                       // x and pos come from the kernels before this one
    const long long t = blockIdx.x, xo = t * a.x_stride, yo = t * a.y_stride;
    const int units = rope_units(VEC, a.rot, a.dim), ty = threadIdx.y, ny = blockDim.y;
    const RopeUnit<VEC> unit(threadIdx.x, a.rot, a.dim, a.interleaved);
    typename RopeUnit<VEC>::Parts p[ROPE_BATCH];
    const int pos = __ldg(a.pos + t);
    rope_fetch(unit, ty, ny, a.heads, a.dim, a.x, a.x_type, xo, p);
    for (int f = ty * blockDim.x + threadIdx.x; f < a.rot >> 1; f += ny * blockDim.x) reinterpret_cast<float2 *>(rope_cs)[f] = rope_angle(pos, __ldg(a.turns + f), a.magnitude);
    __syncthreads();
    rope_put(unit, ty, ny, a.heads, a.dim, a.y, a.y_type, yo, rope_cs, p);
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
        const RopeUnit<VEC> part(u, a.rot, a.dim, a.interleaved);
        for (int h = ty + (u < (int)blockDim.x ? ROPE_BATCH * ny : 0); h < a.heads; h += ROPE_BATCH * ny) {
            rope_fetch(part, h, ny, a.heads, a.dim, a.x, a.x_type, xo, p);
            rope_put(part, h, ny, a.heads, a.dim, a.y, a.y_type, yo, rope_cs, p);
        }
    }
}

extern "C" int ojas_b200_rope_rows(ojas_b200_ctx *ctx, const ojas_b200_rope *rope, int layout, uint32_t x_type, const void *x, size_t x_stride,
                                   uint32_t y_type, void *y, size_t y_stride, const int32_t *pos, size_t M, size_t heads, size_t dim) {
    if (!ctx) return OJAS_B200_E_ARG;
    if (!rope) return ojas_fail(ctx, OJAS_B200_E_ARG, "rope_rows: null rotation");
    if (rope->device != ctx->device) return ojas_fail(ctx, OJAS_B200_E_ARG, "rope_rows: the rotation lives on device %d, the context on %d", rope->device, ctx->device);
    char why[256];
    const int rc = ojas_b200_rope_rows_check(rope->rot_dim, layout, x_type, x, x_stride, y_type, y, y_stride, pos, M, heads, dim, why, sizeof why);
    if (rc) return ojas_fail(ctx, rc, "%s", why);
    if (M == 0) return 0;
    RopeArgs a{};
    a.x = x; a.y = y; a.pos = pos; a.turns = rope->turns; a.magnitude = rope->magnitude;
    a.x_stride = (long long)(x_stride ? x_stride : heads * dim);
    a.y_stride = (long long)(y_stride ? y_stride : heads * dim);
    a.x_type = x_type; a.y_type = y_type;
    a.heads = (int)heads; a.dim = (int)dim; a.rot = (int)rope->rot_dim; a.interleaved = layout == OJAS_B200_ROPE_INTERLEAVED;
    const bool vec = rope_vec_ok(a.rot, a.dim) && rope_rows_aligned(x, x_type, a.x_stride) && rope_rows_aligned(y, y_type, a.y_stride);
    const int units = rope_units(vec ? 4 : 1, a.rot, a.dim);
    const dim3 block(units < 256 ? units : 256, units < 256 ? 256 / units : 1);
    const size_t smem = (size_t)((a.rot / 2 + 1) / 2) * sizeof(float4);
    DeviceGuard guard(ctx->device);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)M); cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, rope_rows_kernel<4>, a) : cudaLaunchKernelEx(&cfg, rope_rows_kernel<1>, a);
    if (e != cudaSuccess) return ojas_fail(ctx, OJAS_B200_E_CUDA, "launch rope_rows: %s", cudaGetErrorString(e));
    OJAS_LAUNCH_CHECK(ctx, "rope_rows");
    return 0;
}

extern "C" int ojas_b200_rope_rows_check(size_t rot_dim, int layout, uint32_t x_type, const void *x, size_t x_stride, uint32_t y_type, const void *y,
                                         size_t y_stride, const int32_t *pos, size_t M, size_t heads, size_t dim, char *err, size_t errlen) {
    auto no = [&](int code, const char *why) { if (err && errlen) snprintf(err, errlen, "rope_rows: %s", why); return code; };
    if (layout != OJAS_B200_ROPE_HALF && layout != OJAS_B200_ROPE_INTERLEAVED) return no(OJAS_B200_E_ARG, "unknown pair layout");
    if (!elem_type(x_type) || !elem_type(y_type)) return no(OJAS_B200_E_ARG, "rows must be f32, f16 or bf16");
    if (heads == 0 || heads > 65536 || dim < 2 || dim > 2048 || dim % 2 != 0) return no(OJAS_B200_E_ARG, "heads must be 1..65536, the head size even, 2..2048");
    if (rot_dim > dim) return no(OJAS_B200_E_ARG, "the rotated part is larger than a head");
    if ((x_stride && x_stride < heads * dim) || (y_stride && y_stride < heads * dim)) return no(OJAS_B200_E_ARG, "a row stride is smaller than a row");
    if (M > 0x3fffffffull || x_stride > (1ull << 40) || y_stride > (1ull << 40)) return no(OJAS_B200_E_LIMIT, "too many rows, or a stride too large");
    if (M && (!x || !y || !pos)) return no(OJAS_B200_E_ARG, "null pointer");
    if (M && ((uintptr_t)x % elem_bytes(x_type) || (uintptr_t)y % elem_bytes(y_type) || (uintptr_t)pos % 4)) return no(OJAS_B200_E_ARG, "a pointer is not aligned to its elements");
    if (M && x == y && (x_type != y_type || (x_stride ? x_stride : heads * dim) != (y_stride ? y_stride : heads * dim)))
        return no(OJAS_B200_E_ARG, "in place, x and y need the same type and stride");
    return 0;
}
