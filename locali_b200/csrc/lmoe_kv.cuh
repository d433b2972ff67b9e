// Shared by the paged key/value cache's kernels (lmoe_kv.cu) and the
// attention over it (lmoe_attn.cu): the cache as the kernels see it, where a
// row's position lives, and the argument structs.
#pragma once

#include "lmoe_common.cuh"

namespace lmoe {

constexpr int kErrIndex = -3;  // LMOE_EINDEX
constexpr int kErrCuda = -4;   // LMOE_ECUDA

// Device view of the cache.  All offsets are 64-bit: a long cache passes 2^31
// elements.
struct KvView {
    uint8_t *kv[2];      // keys, values
    uint16_t *scale[2];  // nullptr when bits is 16
    uint16_t *bias[2];
    int32_t n_pages, page_size, kv_heads;
    uint64_t page_mul;  // ceil(2^(31 + page_shift) / page_size), 2^page_shift >= page_size
    int32_t page_shift;
    // p / page_size for 0 <= p < 2^31: the multiplier is off by less than
    // page_size, so the quotient by less than 1 / page_size
    __device__ __forceinline__ int page_of(int p) const { return (int)((uint64_t)p * page_mul >> (31 + page_shift)); }
    __device__ __forceinline__ int slot_of(int p) const { return p - page_of(p) * page_size; }
    // row index (of head rows) of a slot in a page
    __device__ __forceinline__ int64_t row(int32_t page, int32_t head, int32_t slot) const {
        return ((int64_t)page * kv_heads + head) * page_size + slot;
    }
};

// Positions of a sequence, at most: the end of the key block behind them still
// fits 32 bits (blocks are 128 positions at most).
constexpr int32_t kMaxPos = 0x7FFFFFFF - 255;

struct KvRows {
    const int32_t *table;
    int64_t table_stride;
    int32_t table_width;
    int32_t n_seqs;
    const int32_t *lens;
    const int32_t *row_start;  // nullptr: row b is sequence b's
    int32_t n_rows;
    int32_t max_pos;  // positions a table has room for, kMaxPos at most
    int32_t *err;
    // first row of sequence b, held inside [0, n_rows]
    __device__ __forceinline__ int start(int b) const {
        return row_start ? min(max(row_start[b], 0), n_rows) : b;
    }
    // Threads i of n look through the sequences for lengths and row starts
    // out of range (one block of a launch does).
    __device__ __forceinline__ void validate(int i, int n) const {
        for (int b = i; b < n_seqs; b += n) {
            bool bad = lens[b] < 0 || lens[b] > max_pos;
            if (row_start) bad |= row_start[b] < 0 || row_start[b + 1] < row_start[b] || row_start[b + 1] > n_rows;
            if (bad) set_error(err, kErrIndex);
        }
    }
    // the page that holds position p of sequence b, -1 when it has none
    __device__ __forceinline__ int32_t page(const KvView &c, int b, int p) const {
        const int e = c.page_of(p);
        int32_t pg = -1;
        if (p < max_pos) pg = table[(int64_t)b * table_stride + e];
        if (pg < 0 || pg >= c.n_pages) {
            set_error(err, kErrIndex);
            pg = -1;
        }
        return pg;
    }
};

// Bytes of an attention result, at most (the chunk kernel counts them by 64 in
// 32 bits): more than a B200 holds.
constexpr int64_t kMaxOut = (int64_t)1 << 38;

// packed 16-bit pairs: a b + c, rounded once
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

// packed fp32 pairs
__device__ __forceinline__ uint64_t pack_f2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float &x, float &y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

struct KvCopyArgs {
    KvView c;
    KvRows r;
    const uint16_t *src[2];  // append: new rows
    int64_t tok_stride[2], head_stride[2];
    uint16_t *dst[2];  // read: [n_rows, kv_heads, head_dim]
    int32_t rows_per_block;
};

struct AttnArgs {
    KvView c;
    KvRows r;
    const uint16_t *q;
    int64_t q_tok_stride, q_head_stride;
    uint16_t *out;
    int32_t q_heads;
    int32_t group;  // query heads of one key/value head
    uint64_t group_mul;  // ceil(2^(31 + group_shift) / group), 2^group_shift >= group
    int32_t group_shift;
    float scale_log2;  // scale * log2(e)
    int32_t window, sinks;
    uint8_t *scratch;
    // x / group for 0 <= x < 2^31: the multiplier is off by less than group, so the quotient by less than 1 / group
    __device__ __forceinline__ int per_group(int x) const { return (int)((uint64_t)x * group_mul >> (31 + group_shift)); }
};

cudaError_t launch_attention(int act_f16, int head_dim, int bits, int group_size, const AttnArgs &a, cudaStream_t st);
size_t attention_scratch_bytes(const KvRows &r, int kv_heads, int group, int head_dim);

}  // namespace lmoe
