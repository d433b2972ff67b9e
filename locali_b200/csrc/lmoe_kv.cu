// Paged key/value cache: quantising new rows as they are written, reading
// rows back, and the C entry points of the cache and its attention.
//
// Both kernels move head rows with 16-byte accesses on the 16-bit side: a
// thread owns 8 consecutive elements, head_dim / 8 threads a head row, so a
// group of 32, 64 or 128 elements is 4, 8 or 16 neighbouring lanes and its
// minimum and maximum are a few shuffles.  Every byte moves once; at 31 k rows
// of 8 heads of 128 (B200, launches timed alone): 16 bits, append and read 49
// us each, 5.2 TB/s of the 6.5 a copy reaches; 8-bit groups of 64, read 47 us,
// 4.2 TB/s (a thread's loads are 8 bytes, two in flight), append 90 us, 2.2
// TB/s and bound by issue (about 200 instructions for 8 elements: extremes, the
// scale's division, exact codes; 40 to 60 bytes of spills at five blocks an
// SM); 4 bits, read 49 us, append 95.
#include "../../include/lmoe.h"

#include <cmath>
#include <cstring>

#include "lmoe_kernels.cuh"
#include "lmoe_kv.cuh"

namespace lmoe {

namespace {

constexpr int kKvThreads = 256;
constexpr int kKvMaxRows = 8;  // rows of one block
constexpr int kKvBatch = 2;     // 16-byte pieces of a thread whose loads are in flight together

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

// Scale and bias of a group from its extremes, as 16-bit values; false (both
// NaN) where the group holds an infinity or a NaN.
template <typename TA, int BITS>
__device__ __forceinline__ bool group_scale(float lo, float hi, uint16_t *s16, uint16_t *b16) {
    constexpr float n = (float)((1 << BITS) - 1);
    if (!(fabsf(lo) <= 3.402823466e38f && fabsf(hi) <= 3.402823466e38f)) {
        *s16 = *b16 = Fin<TA>::kNan;
        return false;
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
    return true;
}

// Pairwise maximum of two packed 16-bit pairs, keeping a NaN.
template <typename TA>
__device__ __forceinline__ uint32_t max2_nan(uint32_t x, uint32_t y);
template <>
__device__ __forceinline__ uint32_t max2_nan<__nv_bfloat16>(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}
template <>
__device__ __forceinline__ uint32_t max2_nan<__half>(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}

// Extremes of a group of GS elements, 8 to a lane: the maximum and the
// negated minimum travel as one packed pair.
template <typename TA, int GS>
__device__ __forceinline__ void group_extremes(const uint32_t (&w)[4], float &lo, float &hi) {
    constexpr uint32_t kNeg = 0x80008000u;
    const uint32_t h = max2_nan<TA>(max2_nan<TA>(w[0], w[1]), max2_nan<TA>(w[2], w[3]));
    const uint32_t l = max2_nan<TA>(max2_nan<TA>(w[0] ^ kNeg, w[1] ^ kNeg), max2_nan<TA>(w[2] ^ kNeg, w[3] ^ kNeg));
    uint32_t m = max2_nan<TA>(__byte_perm(h, l, 0x5410), __byte_perm(h, l, 0x7632));
#pragma unroll
    for (int o = 1; o < GS / 8; o <<= 1) m = max2_nan<TA>(m, __shfl_xor_sync(0xffffffffu, m, o));
    hi = Act<TA>::to_f((uint16_t)(m & 0xFFFFu));
    lo = -Act<TA>::to_f((uint16_t)(m >> 16));
}

// Codes clamp(rint((x - b) / s), 0, n) of 8 elements (x >= b), as if computed
// exactly, in the low bytes of q.  (x - b) * (1 / s) in fp32 is within 7e-5
// of the quotient up to 256, 5e-6 up to 16 (2^-24 of the difference, 2^-23 of the approximate
// reciprocal, 2^-24 of the product); only next to a half is the exact side
// needed (0.02 % of elements, but 15 % of warps).  Rounding to an integer is the addition of 1.5 * 2^23,
// whose sum has the code in its low byte.
template <int BITS>
__device__ __forceinline__ void group_codes(const float (&x)[8], float b, float s, uint32_t (&q)[8]) {
    constexpr float n = (float)((1 << BITS) - 1), kMagic = 12582912.0f;
    constexpr float kSure = BITS == 8 ? 0.4999f : 0.49999f;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    const uint64_t nb = pack_f2(-b, -b), i2 = pack_f2(inv, inv), mg = pack_f2(kMagic, kMagic), um = pack_f2(-kMagic, -kMagic);
    const uint64_t neg = pack_f2(-1.0f, -1.0f);
    float off = 0.0f, t[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const uint64_t v = mul_f2(add_f2(pack_f2(x[e], x[e + 1]), nb), i2);
        const uint64_t r = add_f2(v, mg);
        unpack_f2(r, t[e], t[e + 1]);
        float d0, d1;
        unpack_f2(add_f2(v, mul_f2(add_f2(r, um), neg)), d0, d1);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(off) : "f"(fabsf(d0)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(off) : "f"(fabsf(d1)));
    }
    if (!(off < kSure)) {
        if (off <= 0.5f) {
            // The side of the half h: the sign of (x - b) - s h.  x - b is d
            // plus its rounding error, both in fp32; s h (at most 20 bits) and
            // its difference from the near d are exact.
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = x[e] - b, v = d * inv, r = t[e] - kMagic, f = v - r;
                const float bp = d - x[e], err = (x[e] - (d - bp)) + (-b - bp);
                const float low = f > 0.0f ? r : r - 1.0f;
                const float z = fmaf(-s, low + 0.5f, d) + err;
                const float tie = low + ((int)low & 1 ? 1.0f : 0.0f);
                if (!(fabsf(f) < kSure)) t[e] = kMagic + (z == 0.0f ? tie : z > 0.0f ? low + 1.0f : low);
            }
        } else {  // a subnormal or zero scale has no reciprocal
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
                float y = x[0];
#pragma unroll
                for (int k = 1; k < 8; ++k) y = e == k ? x[k] : y;
                y = kMagic + (s > 0.0f ? (float)rint(((double)y - (double)b) / (double)s) : 0.0f);
#pragma unroll
                for (int k = 0; k < 8; ++k) t[k] = e == k ? y : t[k];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __float_as_uint(fminf(t[e], kMagic + n));  // x >= b: no code below 0
}

// where the rows of a block live: page (-1: no place) and slot
struct RowPlace {
    int32_t page, slot;
};

// The first warp finds them: the sequence of the block's first row by
// counting the row starts up to it, 32 at a time (loads that do not wait for
// one another, unlike a binary search's), the other rows from there on.
__device__ __forceinline__ void place_rows(const KvCopyArgs &a, int r0, RowPlace *pl, bool *own) {
    if (blockIdx.x == 0) a.r.validate(threadIdx.x, kKvThreads);
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, r = r0 + lane;
        int b = r;
        if (a.r.row_start) {
            int n = 0;  // row starts at or in front of r0
            for (int b0 = 0; b0 <= a.r.n_seqs; b0 += 32)
                n += __popc(__ballot_sync(0xffffffffu, b0 + lane <= a.r.n_seqs && a.r.start(b0 + lane) <= r0));
            b = max(n - 1, 0);  // none: the first sequence may begin inside the block
        }
        if (lane < a.rows_per_block) {
            RowPlace p{-1, 0};
            bool mine = false;
            if (r < a.r.n_rows) {
                if (a.r.row_start)
                    while (b < a.r.n_seqs && a.r.start(b + 1) <= r) ++b;
                mine = b < a.r.n_seqs && r >= a.r.start(b);  // a row of a sequence, with or without a place
                if (mine) {
                    const int pos = max(a.r.lens[b], 0) - (a.r.start(b + 1) - r);
                    if (pos >= 0) {
                        p.page = a.r.page(a.c, b, pos);
                        p.slot = a.c.slot_of(pos);
                    }
                }
            }
            pl[lane] = p;
            own[lane] = mine;
        }
    }
    __syncthreads();
}

// The pieces of a block's rows in turn: piece i = thread + 256 k is piece
// `u` of row `row` (a row has `units`: keys, then values, by head, 8 elements
// each), walked without a division.
struct Piece {
    int row, u;
    __device__ __forceinline__ Piece(int units) : row(threadIdx.x / units), u(threadIdx.x % units) {}
    __device__ __forceinline__ void step(int units, int dr, int du) {
        row += dr;
        u += du;
        if (u >= units) {
            u -= units;
            ++row;
        }
    }
};

template <typename TA, int BITS, int D, int GS>
__global__ void __launch_bounds__(kKvThreads, 5) kv_append_kernel(const KvCopyArgs a) {
    constexpr int LPR = D / 8;  // lanes of a head row
    constexpr int NG = D / GS;
    __shared__ RowPlace pl[kKvMaxRows];
    __shared__ bool own[kKvMaxRows];
    pdl_wait();
    pdl_trigger();
    const int r0 = blockIdx.x * a.rows_per_block;
    const int units = 2 * a.c.kv_heads * LPR;  // per row
    const int dr = kKvThreads / units, du = kKvThreads % units;
    Piece p(units);
    const int rounds = (a.rows_per_block * units + kKvThreads - 1) / kKvThreads;
    for (int k = 0; k < rounds; k += kKvBatch) {
        uint4 x[kKvBatch];
        Piece at = p;
        auto where = [&](const Piece &q, int &which, int &head, int &c) -> bool {
            const int hv = q.u / LPR;
            c = q.u % LPR;
            which = hv >= a.c.kv_heads;
            head = which ? hv - a.c.kv_heads : hv;
            return q.row < a.rows_per_block && r0 + q.row < a.r.n_rows;
        };
#pragma unroll
        for (int b = 0; b < kKvBatch; ++b) {
            int which, head, c;
            x[b] = make_uint4(0u, 0u, 0u, 0u);
            if (where(p, which, head, c))
                x[b] = *reinterpret_cast<const uint4 *>(a.src[which] + (int64_t)(r0 + p.row) * a.tok_stride[which] +
                                                        (int64_t)head * a.head_stride[which] + c * 8);
            p.step(units, dr, du);
        }
        if (k == 0) place_rows(a, r0, pl, own);  // behind the first loads, which do not need it
#pragma unroll
        for (int b = 0; b < kKvBatch; ++b) {
            int which, head, c;
            // whole head rows are in or out, so the lanes of a group agree
            const bool in = where(at, which, head, c) && pl[at.row].page >= 0;
            if (!__any_sync(0xffffffffu, in)) {  // the rounds' end, rows without a place
                at.step(units, dr, du);
                continue;
            }
            const int64_t row = in ? a.c.row(pl[at.row].page, head, pl[at.row].slot) : 0;
            at.step(units, dr, du);
            if constexpr (BITS == 16) {
                if (in) *reinterpret_cast<uint4 *>(a.c.kv[which] + row * (2 * D) + c * 16) = x[b];
            } else {
                const uint32_t w[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
                float f[8], lo, hi;
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = Act<TA>::to_f((uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu));
                group_extremes<TA, GS>(w, lo, hi);
                uint16_t s16, b16;
                const bool fine = group_scale<TA, BITS>(lo, hi, &s16, &b16);
                uint32_t q[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (fine) group_codes<BITS>(f, lo, Act<TA>::to_f(s16), q);
                if (in) {
                    if constexpr (BITS == 8) {
                        uint2 o;
                        o.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                        o.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
                        *reinterpret_cast<uint2 *>(a.c.kv[which] + row * D + c * 8) = o;
                    } else {
                        // even codes in the low, odd ones in the high nibbles of the bytes
                        const uint32_t ev = __byte_perm(__byte_perm(q[0], q[2], 0x0040), __byte_perm(q[4], q[6], 0x0040), 0x5410);
                        const uint32_t od = __byte_perm(__byte_perm(q[1], q[3], 0x0040), __byte_perm(q[5], q[7], 0x0040), 0x5410);
                        const uint32_t o = ev | od << 4;
                        *reinterpret_cast<uint32_t *>(a.c.kv[which] + row * (D / 2) + c * 4) = o;
                    }
                    if (c % (GS / 8) == 0) {
                        const int64_t gi = row * NG + c / (GS / 8);
                        a.c.scale[which][gi] = s16;
                        a.c.bias[which][gi] = b16;
                    }
                }
            }
        }
    }
}

template <typename TA, int BITS, int D, int GS>
__global__ void __launch_bounds__(kKvThreads, 6) kv_read_kernel(const KvCopyArgs a) {
    constexpr int LPR = D / 8;
    constexpr int NG = D / GS;
    __shared__ RowPlace pl[kKvMaxRows];
    __shared__ bool own[kKvMaxRows];
    pdl_wait();
    pdl_trigger();
    const int r0 = blockIdx.x * a.rows_per_block;
    place_rows(a, r0, pl, own);
    const int units = 2 * a.c.kv_heads * LPR;
    const int dr = kKvThreads / units, du = kKvThreads % units;
    Piece p(units);
    const int rounds = (a.rows_per_block * units + kKvThreads - 1) / kKvThreads;
    for (int k = 0; k < rounds; k += kKvBatch) {
        uint4 o[kKvBatch];  // 16 bits: the row's; else the codes, then scale and bias
        Piece at = p;
#pragma unroll
        for (int b = 0; b < kKvBatch; ++b) {
            o[b] = make_uint4(0u, 0u, 0u, 0u);
            const int hv = p.u / LPR, c = p.u % LPR;
            const int which = hv >= a.c.kv_heads, head = which ? hv - a.c.kv_heads : hv;
            if (p.row < a.rows_per_block && pl[p.row].page >= 0) {
                const int64_t row = a.c.row(pl[p.row].page, head, pl[p.row].slot);
                if constexpr (BITS == 16) {
                    o[b] = *reinterpret_cast<const uint4 *>(a.c.kv[which] + row * (2 * D) + c * 16);
                } else {
                    const int64_t gi = row * NG + c / (GS / 8);
                    if constexpr (BITS == 8) {
                        const uint2 w = *reinterpret_cast<const uint2 *>(a.c.kv[which] + row * D + c * 8);
                        o[b].x = w.x;
                        o[b].y = w.y;
                    } else {
                        o[b].x = *reinterpret_cast<const uint32_t *>(a.c.kv[which] + row * (D / 2) + c * 4);
                    }
                    o[b].z = a.c.scale[which][gi];
                    o[b].w = a.c.bias[which][gi];
                }
            }
            p.step(units, dr, du);
        }
#pragma unroll
        for (int b = 0; b < kKvBatch; ++b) {
            const int hv = at.u / LPR, c = at.u % LPR;
            const int which = hv >= a.c.kv_heads, head = which ? hv - a.c.kv_heads : hv;
            const int row = at.row;
            at.step(units, dr, du);
            if (row >= a.rows_per_block || !own[row]) continue;  // no sequence's row: left as it was
            uint4 v = o[b];
            if constexpr (BITS != 16) {
                // a row without a place: codes, scale and bias 0
                const uint32_t s2 = v.z * 0x10001u, b2 = v.w * 0x10001u;
                uint32_t r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = BITS == 8 ? (e < 2 ? v.x : v.y) >> (16 * (e & 1)) : v.x >> (8 * e);
                    const uint32_t c0 = w & (BITS == 8 ? 255u : 15u), c1 = w >> BITS & (BITS == 8 ? 255u : 15u);
                    r[e] = fma2<TA>(Act<TA>::pack2((float)c0, (float)c1), s2, b2);
                }
                v = make_uint4(r[0], r[1], r[2], r[3]);
            }
            *reinterpret_cast<uint4 *>(a.dst[which] + ((int64_t)(r0 + row) * a.c.kv_heads + head) * D + c * 8) = v;
        }
    }
}

template <typename TA, int BITS, int D, int GS>
cudaError_t launch_kv_t(bool append, KvCopyArgs a, cudaStream_t st) {
    // few rows: one block each, for latency; many: a block takes several, whose look-up (a search, a length and a page
    // id, one behind the other) they share
    a.rows_per_block = a.r.n_rows <= 1024 ? 1 : kKvMaxRows;
    const dim3 grid((unsigned)((a.r.n_rows + a.rows_per_block - 1) / a.rows_per_block));
    return append ? launch_pdl(kv_append_kernel<TA, BITS, D, GS>, grid, dim3(kKvThreads), 0, st, a)
                  : launch_pdl(kv_read_kernel<TA, BITS, D, GS>, grid, dim3(kKvThreads), 0, st, a);
}

template <typename TA>
cudaError_t launch_kv(bool append, int bits, int D, int gs, const KvCopyArgs &a, cudaStream_t st) {
#define LMOE_KV_CASE(B, DD, GG) \
    if (bits == B && D == DD && (B == 16 || gs == GG)) return launch_kv_t<TA, B, DD, GG>(append, a, st);
    LMOE_KV_CASE(16, 64, 64)
    LMOE_KV_CASE(16, 128, 64)
    LMOE_KV_CASE(8, 64, 32)
    LMOE_KV_CASE(8, 64, 64)
    LMOE_KV_CASE(8, 128, 32)
    LMOE_KV_CASE(8, 128, 64)
    LMOE_KV_CASE(8, 128, 128)
    LMOE_KV_CASE(4, 64, 32)
    LMOE_KV_CASE(4, 64, 64)
    LMOE_KV_CASE(4, 128, 32)
    LMOE_KV_CASE(4, 128, 64)
    LMOE_KV_CASE(4, 128, 128)
#undef LMOE_KV_CASE
    return cudaErrorInvalidValue;
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
    }
    v->n_pages = c->n_pages;
    v->page_size = c->page_size;
    while (((int64_t)1 << v->page_shift) < c->page_size) ++v->page_shift;
    v->page_mul = (((uint64_t)1 << (31 + v->page_shift)) + c->page_size - 1) / c->page_size;
    v->kv_heads = c->kv_heads;
    return LMOE_OK;
}

// LMOE_OK with out->n_rows = 0: nothing to do
int check_rows(const lmoe_kv_rows *r, int page_size, void *workspace, KvRows *out) {
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
    const int64_t room = (int64_t)r->table_width * page_size;
    out->max_pos = room < kMaxPos ? (int32_t)room : kMaxPos;
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
    if (!rc) rc = check_rows(rows, cache->page_size, workspace, &a.r);
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
    return kv_rc(cache->dtype == LMOE_F16 ? launch_kv<__half>(true, cache->bits, cache->head_dim, cache->group_size, a, st)
                                          : launch_kv<__nv_bfloat16>(true, cache->bits, cache->head_dim, cache->group_size, a, st));
}

int lmoe_kv_read(const lmoe_kv_cache *cache, const lmoe_kv_rows *rows, void *k, void *v, void *workspace,
                 void *stream) {
    KvCopyArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = check_cache(cache, &a.c);
    if (!rc) rc = check_rows(rows, cache->page_size, workspace, &a.r);
    if (rc || a.r.n_rows == 0) return rc;
    if (!k || !v || !al16(k) || !al16(v)) return LMOE_EINVAL;
    a.dst[0] = static_cast<uint16_t *>(k);
    a.dst[1] = static_cast<uint16_t *>(v);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return kv_rc(cache->dtype == LMOE_F16 ? launch_kv<__half>(false, cache->bits, cache->head_dim, cache->group_size, a, st)
                                          : launch_kv<__nv_bfloat16>(false, cache->bits, cache->head_dim, cache->group_size, a, st));
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
    rc = check_rows(rows, cache->page_size, workspace, &a.r);
    if (rc || a.r.n_rows == 0) return rc;
    if (!strided_ok(q, q_token_stride, q_head_stride) || !out || !al16(out) || !al16(scratch)) return LMOE_EINVAL;
    // row numbers of the tiles (rows x heads of a group) are 32-bit
    if ((int64_t)a.r.n_rows * (q_heads / cache->kv_heads) > (1 << 30)) return LMOE_EUNSUPPORTED;
    if ((int64_t)a.r.n_rows * q_heads * (cache->head_dim * 2) > kMaxOut) return LMOE_EUNSUPPORTED;
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
    // a scale of zero (all terms equal) as the smallest fp32, which no finite score makes visible (2^-149 2^128): 0 times
    // a hidden score's -inf is no number
    a.scale_log2 = fmaxf(scale * 1.4426950408889634f, 1.401298464324817e-45f);
    a.window = window > 0 ? window : 0;
    a.sinks = window > 0 ? sinks : 0;
    a.scratch = static_cast<uint8_t *>(scratch);
    return kv_rc(launch_attention(cache->dtype == LMOE_F16, cache->head_dim, cache->bits, cache->group_size, a,
                                  static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
