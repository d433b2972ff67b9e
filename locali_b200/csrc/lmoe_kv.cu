// Paged key/value cache: quantising new rows as they are written, reading
// rows back, and the C entry points of the cache and its attention.
//
// Both kernels move head rows with 16-byte accesses on the 16-bit side: a
// thread owns 8 consecutive elements, head_dim / 8 threads a head row, so a
// group of 32, 64 or 128 elements is 4, 8 or 16 neighbouring lanes and its
// minimum and maximum are a few shuffles.  Bound by HBM: every byte moves
// once.
#include "../../include/lmoe.h"

#include <cmath>
#include <cstring>

#include "lmoe_kernels.cuh"
#include "lmoe_kv.cuh"

namespace lmoe {

namespace {

constexpr int kKvThreads = 256;
constexpr int kKvMaxRows = 16;  // rows of one block

template <typename TA>
struct Fin;
template <>
struct Fin<__nv_bfloat16> {
    static constexpr float kMax = 3.38953138925153547590470800371487866880e38f;
    static constexpr uint16_t kNan = 0x7FC0;
};
template <>
struct Fin<__half> {
    static constexpr float kMax = 65504.0f;
    static constexpr uint16_t kNan = 0x7E00;
};

template <typename TA>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c);
template <>
__device__ __forceinline__ uint32_t fma2<__nv_bfloat16>(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
template <>
__device__ __forceinline__ uint32_t fma2<__half>(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// Scale and bias of a group from its finite extremes, as 16-bit values.
template <typename TA, int BITS>
__device__ __forceinline__ void group_scale(float lo, float hi, bool bad, uint16_t *s16, uint16_t *b16) {
    constexpr float n = (float)((1 << BITS) - 1);
    if (bad) {
        *s16 = *b16 = Fin<TA>::kNan;
        return;
    }
    // the fp32 quotient is the rounded exact one whenever hi - lo is exact in
    // fp32 (both extremes then reproduce each other); fp64 holds the rest
    const float d = hi - lo;
    float s;
    if (d <= 3.402823466e38f && hi - d == lo && lo + d == hi) s = __fdiv_rn(d, n);
    else s = (float)(((double)hi - (double)lo) / (double)n);
    uint16_t sb = Act<TA>::from_f(s);
    // n codes of the rounded scale may pass the largest finite value
    if (fmaf(Act<TA>::to_f(sb), n, lo) > 0.5f * Fin<TA>::kMax &&
        (double)Act<TA>::to_f(sb) * (double)n + (double)lo > (double)Fin<TA>::kMax)
        sb = (uint16_t)(sb - 1);
    *s16 = sb;
    *b16 = Act<TA>::from_f(lo);
}

// clamp(rint((x - b) / s), 0, n) as if computed exactly.  The fp32 quotient
// is within 5e-5 of the true one up to 255; only next to a half is the exact
// side needed, from fp64.
template <int BITS>
__device__ __forceinline__ uint32_t group_code(float x, float b, float s, float inv) {
    constexpr float n = (float)((1 << BITS) - 1);
    const float q = (x - b) * inv;
    float r = rintf(q);
    if (!(fabsf(q - r) < 0.4999f && q < 1024.0f))
        r = s > 0.0f ? (float)rint(((double)x - (double)b) / (double)s) : 0.0f;
    return (uint32_t)fminf(fmaxf(r, 0.0f), n);
}

// where the rows of a block live: page (-1: no place) and slot
struct RowPlace {
    int32_t page, slot;
};

__device__ __forceinline__ void place_rows(const KvCopyArgs &a, int r0, RowPlace *pl, bool *own) {
    const int i = threadIdx.x;
    if (blockIdx.x == 0) a.r.validate(i, kKvThreads);
    if (i < a.rows_per_block) {
        RowPlace p{-1, 0};
        bool mine = false;
        const int r = r0 + i;
        if (r < a.r.n_rows) {
            int pos = 0;
            const int b = a.r.find(r, &pos);
            mine = b >= 0 || pos < 0;  // a row of a sequence, with or without a place
            if (b >= 0) {
                p.page = a.r.page(a.c, b, pos);
                p.slot = pos % a.c.page_size;
            }
        }
        pl[i] = p;
        own[i] = mine;
    }
    __syncthreads();
}

template <typename TA, int BITS, int D>
__global__ void __launch_bounds__(kKvThreads) kv_append_kernel(const KvCopyArgs a) {
    constexpr int LPR = D / 8;  // lanes of a head row
    __shared__ RowPlace pl[kKvMaxRows];
    __shared__ bool own[kKvMaxRows];
    pdl_wait();
    pdl_trigger();
    const int r0 = blockIdx.x * a.rows_per_block;
    place_rows(a, r0, pl, own);
    const int units = 2 * a.c.kv_heads * LPR;  // per row
    const int total = a.rows_per_block * units;
    for (int i0 = 0; i0 < total; i0 += kKvThreads) {
        const int i = i0 + threadIdx.x;
        // whole head rows are in or out, so the lanes of a group agree
        const int rl = i < total ? i / units : 0;
        const RowPlace p = pl[rl];
        const bool in = i < total && p.page >= 0;
        const int u = i - rl * units;
        const int hv = u / LPR, c = u % LPR;
        const int which = hv >= a.c.kv_heads, head = which ? hv - a.c.kv_heads : hv;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (in)
            x = *reinterpret_cast<const uint4 *>(a.src[which] + (int64_t)(r0 + rl) * a.tok_stride[which] +
                                                 (int64_t)head * a.head_stride[which] + c * 8);
        const int64_t row = in ? a.c.row(p.page, head, p.slot) : 0;
        if constexpr (BITS == 16) {
            if (in) *reinterpret_cast<uint4 *>(a.c.kv[which] + row * (2 * D) + c * 16) = x;
        } else {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = Act<TA>::to_f((uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu));
            float lo = f[0], hi = f[0];
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                lo = fminf(lo, f[e]);
                hi = fmaxf(hi, f[e]);
                bad |= !(fabsf(f[e]) <= 3.402823466e38f);
            }
            uint32_t ibad = bad;
            for (int o = 1; o < a.c.group_size / 8; o <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                ibad |= __shfl_xor_sync(0xffffffffu, ibad, o);
            }
            uint16_t s16, b16;
            group_scale<TA, BITS>(lo, hi, ibad != 0, &s16, &b16);
            const float s = Act<TA>::to_f(s16), b = lo;
            uint32_t q[8];
            const float inv = 1.0f / s;
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = ibad ? 0u : group_code<BITS>(f[e], b, s, inv);
            if (in) {
                if constexpr (BITS == 8) {
                    uint2 o;
                    o.x = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
                    o.y = q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24;
                    *reinterpret_cast<uint2 *>(a.c.kv[which] + row * D + c * 8) = o;
                } else {
                    uint32_t o = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o |= q[e] << (4 * e);
                    *reinterpret_cast<uint32_t *>(a.c.kv[which] + row * (D / 2) + c * 4) = o;
                }
                if (c % (a.c.group_size / 8) == 0) {
                    const int64_t gi = row * a.c.groups + c / (a.c.group_size / 8);
                    a.c.scale[which][gi] = s16;
                    a.c.bias[which][gi] = b16;
                }
            }
        }
    }
}

template <typename TA, int BITS, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const KvCopyArgs a) {
    constexpr int LPR = D / 8;
    __shared__ RowPlace pl[kKvMaxRows];
    __shared__ bool own[kKvMaxRows];
    pdl_wait();
    pdl_trigger();
    const int r0 = blockIdx.x * a.rows_per_block;
    place_rows(a, r0, pl, own);
    const int units = 2 * a.c.kv_heads * LPR;
    const int total = a.rows_per_block * units;
    for (int i = threadIdx.x; i < total; i += kKvThreads) {
        const int rl = i / units;
        if (!own[rl]) continue;  // no sequence's row: left as it was
        const RowPlace p = pl[rl];
        const int u = i - rl * units;
        const int hv = u / LPR, c = u % LPR;
        const int which = hv >= a.c.kv_heads, head = which ? hv - a.c.kv_heads : hv;
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if (p.page >= 0) {
            const int64_t row = a.c.row(p.page, head, p.slot);
            if constexpr (BITS == 16) {
                o = *reinterpret_cast<const uint4 *>(a.c.kv[which] + row * (2 * D) + c * 16);
            } else {
                const int64_t gi = row * a.c.groups + c / (a.c.group_size / 8);
                const uint32_t s2 = a.c.scale[which][gi] * 0x10001u, b2 = a.c.bias[which][gi] * 0x10001u;
                uint32_t r[4];
                if constexpr (BITS == 8) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(a.c.kv[which] + row * D + c * 8);
                    const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t v = ww[e >> 1] >> (16 * (e & 1));
                        r[e] = fma2<TA>(Act<TA>::pack2((float)(v & 255u), (float)(v >> 8 & 255u)), s2, b2);
                    }
                } else {
                    const uint32_t w = *reinterpret_cast<const uint32_t *>(a.c.kv[which] + row * (D / 2) + c * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t v = w >> (8 * e);
                        r[e] = fma2<TA>(Act<TA>::pack2((float)(v & 15u), (float)(v >> 4 & 15u)), s2, b2);
                    }
                }
                o = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
        *reinterpret_cast<uint4 *>(a.dst[which] + ((int64_t)(r0 + rl) * a.c.kv_heads + head) * D + c * 8) = o;
    }
}

template <typename TA, int BITS, int D>
cudaError_t launch_kv_t(bool append, KvCopyArgs a, cudaStream_t st) {
    // few rows: one block each, for latency; many: 8 rows a block
    a.rows_per_block = a.r.n_rows <= 2048 ? 1 : 8;
    const dim3 grid((unsigned)((a.r.n_rows + a.rows_per_block - 1) / a.rows_per_block));
    return append ? launch_pdl(kv_append_kernel<TA, BITS, D>, grid, dim3(kKvThreads), 0, st, a)
                  : launch_pdl(kv_read_kernel<TA, BITS, D>, grid, dim3(kKvThreads), 0, st, a);
}

template <typename TA>
cudaError_t launch_kv(bool append, int bits, int D, const KvCopyArgs &a, cudaStream_t st) {
    if (D == 64) {
        if (bits == 16) return launch_kv_t<TA, 16, 64>(append, a, st);
        if (bits == 8) return launch_kv_t<TA, 8, 64>(append, a, st);
        return launch_kv_t<TA, 4, 64>(append, a, st);
    }
    if (bits == 16) return launch_kv_t<TA, 16, 128>(append, a, st);
    if (bits == 8) return launch_kv_t<TA, 8, 128>(append, a, st);
    return launch_kv_t<TA, 4, 128>(append, a, st);
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_cache(const lmoe_kv_cache *c, KvView *v) {
    if (!c || !c->k || !c->v || c->n_pages < 1 || c->page_size < 1 || c->kv_heads < 1) return LMOE_EINVAL;
    if (c->dtype != LMOE_BF16 && c->dtype != LMOE_F16) return LMOE_EUNSUPPORTED;
    if (c->head_dim != 64 && c->head_dim != 128) return LMOE_EUNSUPPORTED;
    if (c->page_size % 16 != 0 || c->kv_heads > 32767) return LMOE_EUNSUPPORTED;
    const bool quant = c->bits != 16;
    if (quant) {
        if (c->bits != 8 && c->bits != 4) return LMOE_EUNSUPPORTED;
        if ((c->group_size != 32 && c->group_size != 64 && c->group_size != 128) || c->head_dim % c->group_size != 0)
            return LMOE_EUNSUPPORTED;
        if (!c->k_scales || !c->k_biases || !c->v_scales || !c->v_biases) return LMOE_EINVAL;
        if (!al16(c->k_scales) || !al16(c->k_biases) || !al16(c->v_scales) || !al16(c->v_biases)) return LMOE_EINVAL;
    }
    if (!al16(c->k) || !al16(c->v)) return LMOE_EINVAL;
    std::memset(v, 0, sizeof(*v));
    v->kv[0] = static_cast<uint8_t *>(c->k);
    v->kv[1] = static_cast<uint8_t *>(c->v);
    if (quant) {
        v->scale[0] = static_cast<uint16_t *>(c->k_scales);
        v->scale[1] = static_cast<uint16_t *>(c->v_scales);
        v->bias[0] = static_cast<uint16_t *>(c->k_biases);
        v->bias[1] = static_cast<uint16_t *>(c->v_biases);
        v->groups = c->head_dim / c->group_size;
        v->group_size = c->group_size;
    }
    v->n_pages = c->n_pages;
    v->page_size = c->page_size;
    v->kv_heads = c->kv_heads;
    v->row_bytes = c->head_dim * c->bits / 8;
    return LMOE_OK;
}

// LMOE_OK with out->n_rows = 0: nothing to do
int check_rows(const lmoe_kv_rows *r, void *workspace, KvRows *out) {
    if (!r || r->n_seqs < 0 || r->n_rows < 0 || r->table_width < 0 || r->table_stride < r->table_width)
        return LMOE_EINVAL;
    std::memset(out, 0, sizeof(*out));
    if (!r->row_start && r->n_rows != r->n_seqs) return LMOE_EINVAL;
    if (r->n_rows == 0 || r->n_seqs == 0) return LMOE_OK;
    if (!r->lens || (r->table_width > 0 && !r->page_table)) return LMOE_EINVAL;
    out->table = r->page_table;
    out->table_stride = r->table_stride;
    out->table_width = r->table_width;
    out->n_seqs = r->n_seqs;
    out->lens = r->lens;
    out->row_start = r->row_start;
    out->n_rows = r->n_rows;
    out->err = static_cast<int32_t *>(workspace);
    return LMOE_OK;
}

int kv_rc(cudaError_t e) { return e == cudaSuccess ? LMOE_OK : LMOE_ECUDA; }

bool strided_ok(const void *p, int64_t ts, int64_t hs) { return p && al16(p) && ts % 8 == 0 && hs % 8 == 0; }

}  // namespace

}  // namespace lmoe

using namespace lmoe;

extern "C" {

int lmoe_kv_append(const lmoe_kv_cache *cache, const lmoe_kv_rows *rows, const void *k, int64_t k_token_stride,
                   int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride,
                   void *workspace, void *stream) {
    KvCopyArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = check_cache(cache, &a.c);
    if (!rc) rc = check_rows(rows, workspace, &a.r);
    if (rc || a.r.n_rows == 0) return rc;
    if (!strided_ok(k, k_token_stride, k_head_stride) || !strided_ok(v, v_token_stride, v_head_stride))
        return LMOE_EINVAL;
    a.src[0] = static_cast<const uint16_t *>(k);
    a.src[1] = static_cast<const uint16_t *>(v);
    a.tok_stride[0] = k_token_stride;
    a.tok_stride[1] = v_token_stride;
    a.head_stride[0] = k_head_stride;
    a.head_stride[1] = v_head_stride;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return kv_rc(cache->dtype == LMOE_F16 ? launch_kv<__half>(true, cache->bits, cache->head_dim, a, st)
                                          : launch_kv<__nv_bfloat16>(true, cache->bits, cache->head_dim, a, st));
}

int lmoe_kv_read(const lmoe_kv_cache *cache, const lmoe_kv_rows *rows, void *k, void *v, void *workspace,
                 void *stream) {
    KvCopyArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = check_cache(cache, &a.c);
    if (!rc) rc = check_rows(rows, workspace, &a.r);
    if (rc || a.r.n_rows == 0) return rc;
    if (!k || !v || !al16(k) || !al16(v)) return LMOE_EINVAL;
    a.dst[0] = static_cast<uint16_t *>(k);
    a.dst[1] = static_cast<uint16_t *>(v);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return kv_rc(cache->dtype == LMOE_F16 ? launch_kv<__half>(false, cache->bits, cache->head_dim, a, st)
                                          : launch_kv<__nv_bfloat16>(false, cache->bits, cache->head_dim, a, st));
}

size_t lmoe_paged_attention_scratch(const lmoe_kv_cache *cache, const lmoe_kv_rows *rows, int32_t q_heads) {
    KvView c;
    KvRows r;
    if (check_cache(cache, &c) || q_heads < 1 || q_heads % c.kv_heads != 0) return 0;
    if (!rows || rows->n_seqs < 0 || rows->n_rows < 0) return 0;
    std::memset(&r, 0, sizeof(r));
    r.n_seqs = rows->n_seqs;
    r.n_rows = rows->n_rows;
    return attention_scratch_bytes(r, c.kv_heads, q_heads / c.kv_heads, cache->head_dim);
}

int lmoe_paged_attention(const lmoe_kv_cache *cache, const lmoe_kv_rows *rows, int32_t q_heads, const void *q,
                         int64_t q_token_stride, int64_t q_head_stride, float scale, int32_t window, int32_t sinks,
                         void *out, void *scratch, size_t scratch_bytes, void *workspace, void *stream) {
    AttnArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % cache->kv_heads != 0 || sinks < 0) return LMOE_EINVAL;
    if (!(scale >= 0.0f) || scale > 1e30f) return LMOE_EINVAL;
    rc = check_rows(rows, workspace, &a.r);
    if (rc || a.r.n_rows == 0) return rc;
    if (!strided_ok(q, q_token_stride, q_head_stride) || !out || !al16(out) || !al16(scratch)) return LMOE_EINVAL;
    // row numbers of the tiles (rows x heads of a group) are 32-bit
    if ((int64_t)a.r.n_rows * (q_heads / cache->kv_heads) > (1 << 30)) return LMOE_EUNSUPPORTED;
    const size_t need = lmoe_paged_attention_scratch(cache, rows, q_heads);
    if (scratch_bytes < need) return LMOE_EWORKSPACE;
    if (need && !scratch) return LMOE_EINVAL;
    a.q = static_cast<const uint16_t *>(q);
    a.q_tok_stride = q_token_stride;
    a.q_head_stride = q_head_stride;
    a.out = static_cast<uint16_t *>(out);
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    while ((1 << a.group_shift) < a.group) ++a.group_shift;
    a.group_mul = (((uint64_t)1 << (31 + a.group_shift)) + a.group - 1) / a.group;
    // a scale of zero (all terms equal) as one that no score makes visible: 0 times a hidden score's -inf is no number
    a.scale_log2 = fmaxf(scale * 1.4426950408889634f, 2e-38f);
    a.window = window > 0 ? window : 0;
    a.sinks = window > 0 ? sinks : 0;
    a.scratch = static_cast<uint8_t *>(scratch);
    return kv_rc(launch_attention(cache->dtype == LMOE_F16, cache->head_dim, cache->bits, cache->group_size, a,
                                  static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
