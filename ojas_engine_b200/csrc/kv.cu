// The paged key/value cache: its description, the check of a batch on the host, and the append.
//
// A cache is the caller's memory: `pages` pages of page_size tokens for each of `heads` heads of `dim` values, f16 or bf16, with any
// order of the three axes (strides in elements).  A batch says for each sequence which rows of the call are its new tokens
// (cu), how long it is with them (len), and which pages hold it (table).
#include "attn.cuh"
#include "rope.cuh"
#include "tc_util.cuh"

// ---------------------------------------------------------------------------- the cache
static int kv_check(uint32_t type, const void *k, const void *v, size_t pages, size_t page_size, size_t heads, size_t dim, size_t page_stride,
                    size_t head_stride, size_t token_stride, char *err, size_t errlen) {
    auto no = [&](int code, const char *why) { if (err && errlen) snprintf(err, errlen, "kv_create: %s", why); return code; };
    if (type != OJAS_B200_F16 && type != OJAS_B200_BF16) return no(OJAS_B200_E_ARG, "a cache holds f16 or bf16");
    if (dim != 64 && dim != 128 && dim != 256) return no(OJAS_B200_E_UNSUPPORTED, "the head size must be 64, 128 or 256");
    if (page_size == 0 || page_size % 16 != 0) return no(OJAS_B200_E_UNSUPPORTED, "the page size must be a multiple of 16 tokens");
    if (pages == 0 || heads == 0) return no(OJAS_B200_E_ARG, "no pages or no heads");
    if (pages > 0x7fffffffull || page_size > 0x7fffffffull || heads > 65535) return no(OJAS_B200_E_LIMIT, "too many pages, tokens per page or heads");
    if (token_stride < dim || head_stride < dim || (pages > 1 && page_stride < dim)) return no(OJAS_B200_E_ARG, "a stride is smaller than a row");
    if (token_stride % 8 || head_stride % 8 || page_stride % 8) return no(OJAS_B200_E_ARG, "strides must be multiples of 8 elements");
    if (token_stride >= (1ull << 39) || head_stride >= (1ull << 39) || page_stride >= (1ull << 39)) return no(OJAS_B200_E_LIMIT, "a stride is too large");
    // No two rows may share memory: in order of stride, each axis has to step over all that the ones before it span.
    size_t ext[3] = {page_size, heads, pages}, str[3] = {token_stride, head_stride, page_stride};
    for (int i = 0; i < 2; i++)
        for (int j = 0; j < 2 - i; j++)
            if (str[j] > str[j + 1]) {
                size_t t = str[j]; str[j] = str[j + 1]; str[j + 1] = t;
                t = ext[j]; ext[j] = ext[j + 1]; ext[j + 1] = t;
            }
    unsigned __int128 span = dim;
    for (int i = 0; i < 3; i++) {
        if (ext[i] > 1 && str[i] < span) return no(OJAS_B200_E_ARG, "the strides let rows overlap");
        span += (unsigned __int128)(ext[i] - 1) * str[i];
        if (span > ((unsigned __int128)1 << 60)) return no(OJAS_B200_E_LIMIT, "the cache is too large");
    }
    if (!k || !v) return no(OJAS_B200_E_ARG, "null pointer");
    if ((uintptr_t)k % 16 || (uintptr_t)v % 16) return no(OJAS_B200_E_ARG, "the cache must start on 16 bytes");
    return 0;
}

extern "C" int ojas_b200_kv_check(uint32_t type, const void *k, const void *v, size_t pages, size_t page_size, size_t heads, size_t dim,
                                  size_t page_stride, size_t head_stride, size_t token_stride, char *err, size_t errlen) {
    return kv_check(type, k, v, pages, page_size, heads, dim, page_stride, head_stride, token_stride, err, errlen);
}

// Tensor map over one half of the cache: {dim, token in page, head, page}, boxes of 64 values x box_rows tokens that land in
// shared memory as rows of 128 bytes under the 128-byte swizzle.
static int kv_map(ojas_b200_ctx *ctx, const ojas_b200_kv *c, void *base, CUtensorMap *map) {
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return ojas_fail(ctx, OJAS_B200_E_CUDA, "kv_create: cuTensorMapEncodeTiled not found in the driver");
    // An axis of one element may carry any stride; the encoder wants one that is a multiple of 16 bytes.
    const cuuint64_t dims[4] = {c->dim, c->page_size, c->heads, c->pages};
    const cuuint64_t strides[3] = {c->token_stride * 2, c->head_stride * 2, (c->pages > 1 ? c->page_stride : c->dim) * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)c->box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, c->type == OJAS_B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides,
                              box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return ojas_fail(ctx, OJAS_B200_E_CUDA, "kv_create: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return 0;
}

extern "C" int ojas_b200_kv_create(ojas_b200_ctx *ctx, uint32_t type, void *k, void *v, size_t pages, size_t page_size, size_t heads, size_t dim,
                                   size_t page_stride, size_t head_stride, size_t token_stride, ojas_b200_kv **out) {
    if (!ctx || !out) return OJAS_B200_E_ARG;
    *out = nullptr;
    int rc = kv_check(type, k, v, pages, page_size, heads, dim, page_stride, head_stride, token_stride, ctx->err, sizeof ctx->err);
    if (rc) return rc;
    ojas_b200_kv *c = new (std::nothrow) ojas_b200_kv();
    if (!c) return ojas_fail(ctx, OJAS_B200_E_LIMIT, "kv_create: out of host memory");
    c->device = ctx->device; c->type = type; c->k = k; c->v = v;
    c->pages = pages; c->page_size = page_size; c->heads = heads; c->dim = dim;
    c->page_stride = page_stride; c->head_stride = head_stride; c->token_stride = token_stride;
    c->box_rows = 16;
    while (c->box_rows < 64 && page_size % (size_t)(2 * c->box_rows) == 0) c->box_rows *= 2;
    DeviceGuard guard(ctx->device);
    rc = kv_map(ctx, c, k, &c->map_k);
    if (!rc) rc = kv_map(ctx, c, v, &c->map_v);
    if (rc) { delete c; return rc; }
    *out = c;
    return 0;
}

extern "C" void ojas_b200_kv_destroy(ojas_b200_kv *kv) { delete kv; }

// ---------------------------------------------------------------------------- the batch
int seqs_check(const ojas_b200_seqs *s, size_t M, char *err, size_t errlen) {
    auto no = [&](int code, const char *why) { if (err && errlen) snprintf(err, errlen, "sequences: %s", why); return code; };
    if (!s) return no(OJAS_B200_E_ARG, "null pointer");
    if (s->n_seqs > 0x3fffffffull || s->table_stride > 0x7fffffffull || M > 0x3fffffffull) return no(OJAS_B200_E_LIMIT, "too many sequences, pages per sequence or rows");
    if (s->max_rows > 0x3fffffffull || s->max_len > 0x7fffffffull) return no(OJAS_B200_E_LIMIT, "a length bound is too large");
    if (s->n_seqs && M) {
        if (!s->cu || !s->len || !s->table) return no(OJAS_B200_E_ARG, "null pointer");
        if ((uintptr_t)s->cu % 4 || (uintptr_t)s->len % 4 || (uintptr_t)s->table % 4) return no(OJAS_B200_E_ARG, "a pointer is not aligned to its elements");
        if (s->table_stride == 0) return no(OJAS_B200_E_ARG, "a page table without entries");
        if (s->max_rows == 0 || s->max_len == 0) return no(OJAS_B200_E_ARG, "max_rows and max_len bound the sequences' new rows and lengths: both at least 1");
    }
    return 0;
}

extern "C" int ojas_b200_seqs_check_host(const int32_t *cu, const int32_t *len, const int32_t *table, size_t n_seqs, size_t table_stride, size_t max_rows,
                                         size_t max_len, size_t pages, size_t page_size, size_t M, char *err, size_t errlen) {
    auto no = [&](size_t b, const char *why) { if (err && errlen) snprintf(err, errlen, "sequence %zu: %s", b, why); return OJAS_B200_E_ARG; };
    if (!cu || (n_seqs && (!len || !table)) || page_size == 0) return no(0, "null pointer or no page size");
    if (cu[0] < 0) return no(0, "its rows begin before the call's first");
    for (size_t b = 0; b < n_seqs; b++) {
        if (cu[b + 1] < cu[b]) return no(b, "its rows end before they begin");
        if ((size_t)cu[b + 1] > M) return no(b, "its rows end behind the call's last");
        const size_t rows = (size_t)(cu[b + 1] - cu[b]);
        if (rows > max_rows) return no(b, "more new rows than max_rows");
        if (len[b] < 0 || (size_t)len[b] < rows) return no(b, "shorter than its new rows");
        if ((size_t)len[b] > max_len) return no(b, "longer than max_len");
        const size_t used = ((size_t)len[b] + page_size - 1) / page_size;
        if (used > table_stride) return no(b, "longer than its pages");
        for (size_t i = 0; i < used; i++)
            if (table[b * table_stride + i] < 0 || (size_t)table[b * table_stride + i] >= pages) return no(b, "a page number outside the cache");
    }
    return 0;
}

// ---------------------------------------------------------------------------- append
// One head row of the call: read, rotated (q, k) or not (v), rounded to its destination's type, written once.  HBM bound: the
// bytes of q, k and v in, of q_out and the cache rows out.
struct AppendArgs {
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    const int *pos;                    // null: a token's place in its sequence
    const uint64_t *turns;             // null: no rotation
    float magnitude;
    long long q_stride, k_stride, v_stride, q_out_stride, page_stride, head_stride, token_stride;
    BatchArgs batch;
    uint32_t x_type, q_type, c_type;
    int q_heads, kv_heads, dim, rot;
    bool interleaved;
};

// One CTA per token, as rope_rows: the first loads of q, k and v go out before the token's place is looked up.
template <int VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendArgs a) {
    extern __shared__ float4 append_cs[];                // (cos, sin) of two pairs each
    __shared__ long long row_at_s;                       // element offset of the token's row of head 0 in the cache; -1: not written
    __shared__ int row_pos_s;                            // position of rotation
    __shared__ bool row_live_s;                          // the row belongs to a sequence
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const long long t = blockIdx.x;
    const int rot = a.turns ? a.rot : 0, units = rope_units(VEC, rot, a.dim);
    const int ux = threadIdx.x % units, uy = threadIdx.x / units, ny = blockDim.x / units;   // (dim <= 256: at most 128 units)
    const RopeUnit<VEC> unit(uy < ny ? ux : units, rot, a.dim, a.interleaved), plain(uy < ny ? ux : units, 0, a.dim, false);   // (a thread too many has nothing)
    typename RopeUnit<VEC>::Parts p[ROPE_BATCH], k, v;
    const long long qo = t * a.q_stride, ko = t * a.k_stride, vo = t * a.v_stride;
    rope_fetch(unit, uy, ny, a.q_heads, a.dim, a.q, a.x_type, qo, p);
    if (uy < a.kv_heads) {
        unit.fetch(a.k, a.x_type, ko + uy * a.dim, k);
        plain.fetch(a.v, a.x_type, vo + uy * a.dim, v);
    }
    if (threadIdx.x < 32) {
        const int b = find_seq(a.batch.cu, a.batch.n_seqs, t, lane);
        if (lane == 0) {
            long long at = -1;
            int pos = 0;
            if (b >= 0) {
                const int first = __ldg(a.batch.cu + b), end = __ldg(a.batch.cu + b + 1);
                const long long at_pos = (long long)__ldg(a.batch.len + b) - end + t;      // = len - rows + (t - first)
                const long long entry = at_pos / a.batch.page_size;
                int page = -1;
                if (at_pos >= 0 && first >= 0 && entry < a.batch.table_stride) page = __ldg(a.batch.table + (long long)b * a.batch.table_stride + entry);
                if (page >= 0 && page < a.batch.pages) at = (long long)page * a.page_stride + (at_pos - entry * a.batch.page_size) * a.token_stride;
                else atomicOr(a.batch.status, OJAS_ST_BATCH);                              // nowhere to put it: q is still turned
                pos = a.pos ? __ldg(a.pos + t) : (int)at_pos;
            }
            row_live_s = b >= 0;
            row_at_s = at;
            row_pos_s = pos;
        }
    }
    // The second warp looks at the offsets themselves, a share of them per CTA: rows outside the call have no CTA of their own.
    if (threadIdx.x >> 5 == 1) {
        for (long long b = t * 32 + lane; b < a.batch.n_seqs; b += a.batch.M * 32)
            if (!seq_in_call(__ldg(a.batch.cu + b), __ldg(a.batch.cu + b + 1), a.batch.M)) atomicOr(a.batch.status, OJAS_ST_BATCH);
    }
    __syncthreads();
    if (!row_live_s) return;
    for (int f = threadIdx.x; f < rot >> 1; f += blockDim.x) reinterpret_cast<float2 *>(append_cs)[f] = rope_angle(row_pos_s, __ldg(a.turns + f), a.magnitude);
    __syncthreads();
    const long long row_at = row_at_s, q_to = t * a.q_out_stride;
    if (row_at >= 0) {
        for (int h = uy; h < a.kv_heads; h += ny) {
            if (h != uy) {
                unit.fetch(a.k, a.x_type, ko + h * a.dim, k);
                plain.fetch(a.v, a.x_type, vo + h * a.dim, v);
            }
            unit.put(k, a.kc, a.c_type, row_at + (long long)h * a.head_stride, append_cs);
            plain.put(v, a.vc, a.c_type, row_at + (long long)h * a.head_stride, append_cs);
        }
    }
    rope_put(unit, uy, ny, a.q_heads, a.dim, a.q_out, a.q_type, q_to, append_cs, p);
    for (int h = uy + ROPE_BATCH * ny; h < a.q_heads; h += ROPE_BATCH * ny) {
        rope_fetch(unit, h, ny, a.q_heads, a.dim, a.q, a.x_type, qo, p);
        rope_put(unit, h, ny, a.q_heads, a.dim, a.q_out, a.q_type, q_to, append_cs, p);
    }
}

static int append_check(size_t kv_heads, size_t dim, size_t rot, int layout, uint32_t x_type, const void *q, size_t q_stride, const void *k, size_t k_stride,
                        const void *v, size_t v_stride, uint32_t q_type, const void *q_out, size_t q_out_stride, size_t q_heads, const int32_t *pos,
                        size_t M, char *err, size_t errlen) {
    auto no = [&](int code, const char *why) { if (err && errlen) snprintf(err, errlen, "kv_append: %s", why); return code; };
    if (!elem_type(x_type)) return no(OJAS_B200_E_ARG, "rows must be f32, f16 or bf16");
    if (rot && layout != OJAS_B200_ROPE_HALF && layout != OJAS_B200_ROPE_INTERLEAVED) return no(OJAS_B200_E_ARG, "unknown pair layout");
    if (rot > dim) return no(OJAS_B200_E_ARG, "the rotated part is larger than a head");
    if (q_heads > 65536) return no(OJAS_B200_E_LIMIT, "more than 65536 query heads");
    if ((k_stride && k_stride < kv_heads * dim) || (v_stride && v_stride < kv_heads * dim)) return no(OJAS_B200_E_ARG, "a row stride is smaller than a row");
    if (k_stride > (1ull << 40) || v_stride > (1ull << 40) || q_stride > (1ull << 40) || q_out_stride > (1ull << 40)) return no(OJAS_B200_E_LIMIT, "a stride is too large");
    if (M && (!k || !v)) return no(OJAS_B200_E_ARG, "null pointer");
    if (M && ((uintptr_t)k % elem_bytes(x_type) || (uintptr_t)v % elem_bytes(x_type) || (uintptr_t)pos % 4)) return no(OJAS_B200_E_ARG, "a pointer is not aligned to its elements");
    if (q_heads) {
        if (!elem_type(q_type)) return no(OJAS_B200_E_ARG, "q_out must be f32, f16 or bf16");
        if ((q_stride && q_stride < q_heads * dim) || (q_out_stride && q_out_stride < q_heads * dim)) return no(OJAS_B200_E_ARG, "a row stride is smaller than a row");
        if (M && (!q || !q_out)) return no(OJAS_B200_E_ARG, "query heads without q and q_out");
        if (M && ((uintptr_t)q % elem_bytes(x_type) || (uintptr_t)q_out % elem_bytes(q_type))) return no(OJAS_B200_E_ARG, "a pointer is not aligned to its elements");
        if (M && q == q_out && (x_type != q_type || (q_stride ? q_stride : q_heads * dim) != (q_out_stride ? q_out_stride : q_heads * dim)))
            return no(OJAS_B200_E_ARG, "in place, q and q_out need the same type and stride");
    }
    return 0;
}

extern "C" int ojas_b200_kv_append_check(size_t kv_heads, size_t dim, size_t rot_dim, int layout, uint32_t x_type, const void *q, size_t q_stride,
                                         const void *k, size_t k_stride, const void *v, size_t v_stride, uint32_t q_type, const void *q_out,
                                         size_t q_out_stride, size_t q_heads, const int32_t *pos, const ojas_b200_seqs *seqs, size_t M, char *err,
                                         size_t errlen) {
    const int rc = append_check(kv_heads, dim, rot_dim, layout, x_type, q, q_stride, k, k_stride, v, v_stride, q_type, q_out, q_out_stride, q_heads, pos, M, err, errlen);
    return rc ? rc : seqs_check(seqs, M, err, errlen);
}

extern "C" int ojas_b200_kv_append(ojas_b200_ctx *ctx, const ojas_b200_kv *kv, const ojas_b200_seqs *seqs, const ojas_b200_rope *rope, int layout,
                                   uint32_t x_type, const void *q, size_t q_stride, const void *k, size_t k_stride, const void *v, size_t v_stride,
                                   uint32_t q_type, void *q_out, size_t q_out_stride, size_t q_heads, const int32_t *pos, size_t M) {
    if (!ctx) return OJAS_B200_E_ARG;
    if (!kv) return ojas_fail(ctx, OJAS_B200_E_ARG, "kv_append: null cache");
    if (kv->device != ctx->device || (rope && rope->device != ctx->device))
        return ojas_fail(ctx, OJAS_B200_E_ARG, "kv_append: the cache or the rotation lives on another device than the context's (%d)", ctx->device);
    char why[256];
    const int rc = ojas_b200_kv_append_check(kv->heads, kv->dim, rope ? rope->rot_dim : 0, layout, x_type, q, q_stride, k, k_stride, v, v_stride, q_type, q_out,
                                             q_out_stride, q_heads, pos, seqs, M, why, sizeof why);
    if (rc) return ojas_fail(ctx, rc, "%s", why);
    if (M == 0 || seqs->n_seqs == 0) return 0;
    AppendArgs a{};
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.kc = kv->k; a.vc = kv->v; a.pos = pos;
    a.turns = rope ? rope->turns : nullptr; a.magnitude = rope ? rope->magnitude : 1.0f; a.rot = rope ? (int)rope->rot_dim : 0;
    a.interleaved = layout == OJAS_B200_ROPE_INTERLEAVED;
    a.q_stride = (long long)(q_stride ? q_stride : q_heads * kv->dim);
    a.q_out_stride = (long long)(q_out_stride ? q_out_stride : q_heads * kv->dim);
    a.k_stride = (long long)(k_stride ? k_stride : kv->heads * kv->dim);
    a.v_stride = (long long)(v_stride ? v_stride : kv->heads * kv->dim);
    a.page_stride = (long long)kv->page_stride; a.head_stride = (long long)kv->head_stride; a.token_stride = (long long)kv->token_stride;
    a.batch = {seqs->cu, seqs->len, seqs->table, (int)seqs->n_seqs, (int)seqs->table_stride, (long long)M, (int)kv->pages, (int)kv->page_size, (int)seqs->max_rows, ctx->dev_status};
    a.x_type = x_type; a.q_type = q_type; a.c_type = kv->type;
    a.q_heads = (int)q_heads; a.kv_heads = (int)kv->heads; a.dim = (int)kv->dim;
    const bool vec = rope_vec_ok(a.rot, a.dim) && rope_rows_aligned(k, x_type, a.k_stride) && rope_rows_aligned(v, x_type, a.v_stride) &&
                     (q_heads == 0 || (rope_rows_aligned(q, x_type, a.q_stride) && rope_rows_aligned(q_out, q_type, a.q_out_stride)));
    const size_t smem = (size_t)((a.rot / 2 + 1) / 2) * sizeof(float4);
    DeviceGuard guard(ctx->device);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)M); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = smem; cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, kv_append_kernel<4>, a) : cudaLaunchKernelEx(&cfg, kv_append_kernel<1>, a);
    if (e != cudaSuccess) return ojas_fail(ctx, OJAS_B200_E_CUDA, "launch kv_append: %s", cudaGetErrorString(e));
    OJAS_LAUNCH_CHECK(ctx, "kv_append");
    return 0;
}
