// Shared by the attention kernels: which keys a tile of rows sees, how the
// work of a launch is cut over its blocks, and 16-bit pair arithmetic.
#pragma once

#include "lmoe_kernels.cuh"
#include "lmoe_kv.cuh"

namespace lmoe {

// A tile is up to R consecutive rows of one sequence for one key/value head,
// where the rows of a sequence are its tokens times the group's query heads
// (row i = token i / group, head i % group).  Its keys are walked in blocks
// of KS positions: first the blocks of the first tokens that stay visible
// (sinks), then the blocks from the window's lower edge of its first token to
// its last token's position.
struct Tile {
    int b, rt, h;       // sequence, row tile, key/value head
    int row0;           // first row of the arrays that is the sequence's
    int n;              // its token rows
    int first;          // position of its token row 0 (may be negative)
    int rows;           // rows of the tile, 1..R
    int minpos, maxpos; // positions of the tile's first and last row
    int hi;             // keys [0, hi) are looked at: those the table has room for
    int nsink, lo;      // sink blocks, first block of the rest (held at the first one behind hi)
    int nblk;           // blocks; at least 1, so a tile that sees nothing is written
    __device__ __forceinline__ int block(int i) const { return i < nsink ? i : lo + i - nsink; }
};

template <int R, int KS>
__device__ __forceinline__ void tile_range(const AttnArgs &a, Tile &t) {
    const int r0 = t.rt * R;
    t.rows = min(R, t.n * a.group - r0);
    t.minpos = t.first + a.per_group(r0);
    t.maxpos = t.first + a.per_group(r0 + t.rows - 1);
    t.hi = min(max(0, t.maxpos + 1), a.r.max_pos);
    int low = 0;
    if (a.window > 0) low = (int)max(0ll, (long long)t.minpos - a.window + 1);
    // Held at the first block behind hi: the window of a length far past its
    // table may begin in the last block that 32 bits can count, whose end they
    // cannot.
    t.lo = min(low / KS, (t.hi + KS - 1) / KS);
    t.nsink = t.lo > 0 ? min((min(a.sinks, t.hi) + KS - 1) / KS, t.lo) : 0;
    t.nblk = max(1, t.nsink + max(0, (t.hi + KS - 1) / KS - t.lo));
}

// Does a row of the tile see one of the 16 positions from p < hi?  Blocks
// reach past the first tokens and the window's lower edge, and what lies
// between those may have no page any more.  (In numbers the tile holds anyway:
// one more cost registers and 3 % of the few-row kernel.)
__device__ __forceinline__ bool run_seen(const AttnArgs &a, const Tile &t, int p) {
    return a.window == 0 || t.minpos - p - 15 < a.window || p < a.sinks;
}

// Sequence b's rows into t; returns its tiles (of one head).
template <int R>
__device__ __forceinline__ int seq_rows(const AttnArgs &a, int b, Tile &t) {
    t.b = b;
    t.row0 = a.r.start(b);
    t.n = max(0, a.r.start(b + 1) - t.row0);
    t.first = max(a.r.lens[b], 0) - t.n;
    return (t.n * a.group + R - 1) / R;
}

// The work of a launch is a stream: for every (sequence, row tile, head), in
// that order, X units for the tile itself (its rows, its result) and one for
// each key block.  Block c of the launch takes the c-th of `parts` equal runs
// of it.  So ragged batches stay level without the host knowing a length, and
// a tile may be cut over several blocks of the launch; attn_merge_kernel joins
// those.
// quotient of values that mostly fit 32 bits
__device__ __forceinline__ long long div_small(long long x, long long y) {
    return ((x | y) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)y) : x / y;
}
struct Share {
    long long total;  // units of the stream
    long long each;   // a run's units; the first `more` runs have one more
    int parts;        // launch blocks that take part
    int more;
    __device__ __forceinline__ void split(long long units, int n) {
        total = units;
        parts = n;
        each = div_small(units, n);
        more = (int)(units - each * n);
    }
    __device__ __forceinline__ long long begin(int c) const { return each * c + min(c, more); }
    __device__ __forceinline__ int owner(long long x) const {
        const long long big = (each + 1) * more;
        return x < big ? (int)div_small(x, each + 1) : more + (int)div_small(x - big, each);
    }
};

// A run's place in the stream: the tile, where the stream has its first unit,
// and the key blocks [b0, b1) of it that are the run's (none: b0 == b1).
template <int R, int KS, int X>
struct Cursor {
    Tile t;
    long long at, end;  // the tile's first unit, the run's end
    int b0, b1;
    __device__ __forceinline__ void open(long long from) {
        b0 = (int)max(0ll, from - at - X);
        b1 = (int)max((long long)b0, min((long long)t.nblk, end - at - X));
    }
    // launch blocks that share the tile, if it begins here and goes on behind the run; else 0
    __device__ __forceinline__ int shared(const Share &sh, int c) const {
        return b0 == 0 && b1 > 0 && b1 < t.nblk ? sh.owner(at + X + t.nblk - 1) - c + 1 : 0;
    }
    // The next tile with key blocks of the run's; false: there is none.
    __device__ __forceinline__ bool next(const AttnArgs &a) {
        for (;;) {
            at += X + t.nblk;
            if (at + X >= end) return false;
            if (++t.h >= a.c.kv_heads) {
                t.h = 0;
                if (++t.rt * (long long)R >= (long long)t.n * a.group) {
                    t.rt = 0;
                    int b = t.b, nt;
                    do {
                        if (++b >= a.r.n_seqs) return false;
                        nt = seq_rows<R>(a, b, t);
                    } while (nt == 0);
                }
                tile_range<R, KS>(a, t);
            }
            open(at);
            if (b1 > b0) return true;
        }
    }
};

// Units of sequence b for one head.  A thread walks its tiles, or (WARP) a
// warp's lanes share them; all lanes then hold the sum.
template <int R, int KS, int X, bool WARP>
__device__ __forceinline__ long long seq_units(const AttnArgs &a, int b) {
    Tile t;
    const int nt = seq_rows<R>(a, b, t);
    long long sum = 0;
    for (t.rt = WARP ? (threadIdx.x & 31) : 0; t.rt < nt; t.rt += WARP ? 32 : 1) {
        tile_range<R, KS>(a, t);
        sum += t.nblk + X;
    }
    if (WARP) {
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    return sum;
}

// Finds the launch block's run; every thread of the block calls it (NTHR
// threads, sm of NTHR / 32 + 4 long longs).  False: no work.  WARP: a warp for
// each sequence (few sequences of many tiles), else a thread.  minu: units a
// run has at least.  Lengths and row starts are read more than once and must
// not change meanwhile; no search here or in Cursor::next rests its end on
// that.
template <int R, int KS, int X, int NTHR, bool WARP>
__device__ __forceinline__ bool find_share(const AttnArgs &a, int minu, long long *sm, Share &sh, Cursor<R, KS, X> &cur) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = NTHR / 32, PER = WARP ? NW : NTHR;  // sequences of a round
    const int rounds = (a.r.n_seqs + PER - 1) / PER;
    auto units = [&](int k) -> long long {  // of this warp's or thread's sequence of round k
        const int b = k * PER + (WARP ? warp : tid);
        return b < a.r.n_seqs ? seq_units<R, KS, X, WARP>(a, b) * a.c.kv_heads : 0;
    };
    const long long mine = units(0);
    long long sum = mine;
    for (int k = 1; k < rounds; ++k) sum += units(k);
    if (!WARP) {
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) sm[warp] = sum;
    if (tid < 4) sm[NW + tid] = 0;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < NW; ++w) total += sm[w];
    __syncthreads();
    if (total == 0) return false;
    sh.split(total, (int)min((long long)gridDim.x, max(1ll, div_small(total, minu))));
    if ((int)blockIdx.x >= sh.parts) return false;
    const long long s = sh.begin(blockIdx.x);
    // the sequence that holds unit s
    long long base = 0;
    for (int k = 0; k < rounds; ++k) {
        const long long w = k == 0 ? mine : units(k);
        long long inc = w;
        if (!WARP) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
        }
        if (lane == 31) sm[warp] = inc;
        __syncthreads();
        long long before = base;
        for (int q = 0; q < NW; ++q) {
            if (q < warp) before += sm[q];
            base += sm[q];
        }
        before += inc - w;
        if (w > 0 && before <= s && s < before + w && (!WARP || lane == 0)) {
            sm[NW] = k * PER + (WARP ? warp : tid);
            sm[NW + 1] = before;
        }
        __syncthreads();
        if (s < base) break;
    }
    // its tile: the first warp's lanes look at 32 tiles at a time
    Tile &t = cur.t;
    const int nt = seq_rows<R>(a, (int)sm[NW], t);
    if (warp == 0) {
        long long off = s - sm[NW + 1];
        for (int r0 = 0; r0 < nt; r0 += 32) {
            t.rt = r0 + lane;
            long long w = 0;
            if (t.rt < nt) {
                tile_range<R, KS>(a, t);
                w = (long long)(t.nblk + X) * a.c.kv_heads;
            }
            long long inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, off < inc);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    sm[NW + 2] = t.rt;
                    sm[NW + 3] = off - (inc - w);
                }
                break;
            }
            off -= __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    __syncthreads();
    t.rt = (int)sm[NW + 2];
    tile_range<R, KS>(a, t);
    const long long off = sm[NW + 3];
    t.h = min((int)div_small(off, t.nblk + X), a.c.kv_heads - 1);
    cur.at = s - (off - (long long)t.h * (t.nblk + X));
    cur.end = sh.begin(blockIdx.x + 1);
    cur.open(s);
    __syncthreads();
    return cur.b1 > cur.b0 || cur.next(a);
}

// Scratch: one record for each launch block (the cut tile that begins in its
// run, if any), then two partial results each: slot 0 of a launch block is
// its part of a tile begun before it, slot 1 of the tile that goes on behind
// it.  A partial: R rows of D fp32 sums, then R (maximum, sum) pairs.
struct MergeRec {
    int32_t parts;  // 0 or 1: nothing to merge
    int32_t out0;   // first row of the sequence
    int32_t row;    // first row of the tile in the sequence's rows
    int32_t rows_h; // rows | head << 16
};
template <int R, int D>
__host__ __device__ constexpr size_t part_floats() {
    return (size_t)R * (D + 2);
}
__device__ __forceinline__ float *part_ptr(const AttnArgs &a, int grid, size_t floats, int c, int slot) {
    return reinterpret_cast<float *>(a.scratch + (size_t)grid * sizeof(MergeRec)) + ((size_t)2 * c + slot) * floats;
}

// A row's terms are exp2(score - m), m its reference: any value may serve, as
// the result is a quotient.  m is set so that the largest score's term is
// 2^kSet.  The few-row kernel sets it at every larger score.  The chunk kernel,
// whose sums lie in tensor memory, waits until a term would pass 2^kTop (2^8
// above; 2^4 for f16, set 2^11 high, cost windowed chunks 15 %).
//   f16: the terms of many keys far below the largest still count together,
//   and f16 has no normal value under 2^-14: the largest term is put near the
//   largest f16, so terms of 2^-29 of it (chunks: 2^-21) and more keep all
//   their bits.
//   bf16: a value may be near 2^128, where the fp32 sums end too: with terms of
//   2^-24 (2^-16) the sums of 2^16 keys and more stay below it.  The price is
//   at the other end, where values under 2^-100 lose bits.
template <typename TA, bool CHUNK>
struct Term {
    static constexpr bool kF16 = std::is_same<TA, __half>::value;
    static constexpr float kSet = kF16 ? (CHUNK ? 7.0f : 15.0f) : -24.0f;
    static constexpr float kTop = kF16 ? 15.0f : -16.0f;
};

// 16 bytes into shared memory, `bytes` of them from src and zeros behind
__device__ __forceinline__ void cp16z(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ------------------------------------------------------------ packed 16-bit pairs
template <typename TA>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
    __device__ __forceinline__ static uint32_t fma(uint32_t a, uint32_t b, uint32_t c) { return fma2<__nv_bfloat16>(a, b, c); }
    __device__ __forceinline__ static uint32_t mul(uint32_t a, uint32_t b) { return fma(a, b, 0x80008000u); }
    // 8-bit codes: the code's bits are a bf16 subnormal, c * 2^-133;
    // multiplied by 2^127 it is c * 2^-6 exactly, and the scale is taken times
    // 2^6 (exact, no overflow: a scale is at most 2^129 / 255).  4-bit codes,
    // whose scales may be larger: 0x4300 | c is 128 + c.
    template <int BITS>
    __device__ __forceinline__ static uint32_t scale(uint32_t s2) {
        return BITS == 8 ? mul(s2, 0x42804280u) : s2;
    }
    __device__ __forceinline__ static uint32_t value8(uint32_t c, uint32_t s2, uint32_t b2) {
        return fma(mul(c, 0x7F007F00u), s2, b2);
    }
    // code j of each half
    __device__ __forceinline__ static uint32_t value4(uint32_t u, int j, uint32_t s2, uint32_t b2) {
        return fma(fma(and_or(u >> (4 * j), 0x000F000Fu, 0x43004300u), 0x3F803F80u, 0xC300C300u), s2, b2);
    }
    static constexpr uint32_t kExpMask = 0x7F80u;
};
template <>
struct Pair<__half> {
    __device__ __forceinline__ static uint32_t fma(uint32_t a, uint32_t b, uint32_t c) { return fma2<__half>(a, b, c); }
    template <int BITS>
    __device__ __forceinline__ static uint32_t scale(uint32_t s2) {
        return s2;
    }
    // 0x6400 | c is 1024 + c
    __device__ __forceinline__ static uint32_t value8(uint32_t c, uint32_t s2, uint32_t b2) {
        return fma(fma(c | 0x64006400u, 0x3C003C00u, 0xE400E400u), s2, b2);
    }
    // code j of each half; at bits 4..7, 0x6400 | c << 4 is 1024 + 16 c
    __device__ __forceinline__ static uint32_t value4(uint32_t u, int j, uint32_t s2, uint32_t b2) {
        const uint32_t v = j < 2 ? u : u >> 8;
        return j & 1 ? fma(fma(and_or(v, 0x00F000F0u, 0x64006400u), 0x2C002C00u, 0xD400D400u), s2, b2)
                     : fma(fma(and_or(v, 0x000F000Fu, 0x64006400u), 0x3C003C00u, 0xE400E400u), s2, b2);
    }
    static constexpr uint32_t kExpMask = 0x7C00u;
};

// Pair j of a word's two halves as an operand without scale and bias, (code +
// kOffset) kUnit: what the cheapest way to a number gives (j = 0..3 for 4-bit
// codes, 0..1 for 8-bit ones).  Scores are summed times kDown: a bf16 scale of
// 4-bit codes may be 2^125, and 128 of those are no fp32 (8 bits down they
// are, and the smallest scale and bias stay exact; the codes are put there by
// their exponent, so the scale needs no multiplication).
template <typename TA, int BITS>
struct RawCode {
    static constexpr bool kBf = std::is_same<TA, __nv_bfloat16>::value;
    static constexpr float kOffset = kBf ? (BITS == 8 ? 0.0f : 128.0f) : 1024.0f;
    static constexpr float kUnit = kBf ? (BITS == 8 ? 1.0f / 64.0f : 1.0f / 256.0f) : 1.0f;
    static constexpr float kDown = kBf && BITS == 4 ? 1.0f / 256.0f : 1.0f;
    __device__ __forceinline__ static uint32_t pair(uint32_t u, int j) {
        if constexpr (BITS == 4) return and_or(u >> (4 * j), 0x000F000Fu, kBf ? 0x3F003F00u : 0x64006400u);
        else if constexpr (kBf) return Pair<TA>::mul(j ? __byte_perm(u, 0u, 0x4341) : u & 0x00FF00FFu, 0x7F007F00u);
        else return j ? __byte_perm(u, 0x64646464u, 0x4341) : and_or(u, 0x00FF00FFu, 0x64006400u);
    }
};

// Value pair j of a word's two halves: 4-bit codes j = 0..3, 8-bit codes j = 0..1.
template <typename TA, int BITS>
__device__ __forceinline__ uint32_t code_pair(uint32_t u, int j, uint32_t s2, uint32_t b2) {
    if constexpr (BITS == 4) return Pair<TA>::value4(u, j, s2, b2);
    else return Pair<TA>::value8(j ? __byte_perm(u, 0u, 0x4341) : u & 0x00FF00FFu, s2, b2);
}

template <typename TA>
__device__ __forceinline__ bool nonfinite16(uint32_t x) {
    return (x & Pair<TA>::kExpMask) == Pair<TA>::kExpMask;
}
// The value of one code before its rounding; like the pairs above no number
// for bf16 scales of 8-bit codes from 2^122 on.
template <typename TA, int BITS>
__device__ __forceinline__ float code_value(uint32_t code, uint32_t s16, uint32_t b16) {
    constexpr float up = std::is_same<TA, __nv_bfloat16>::value && BITS == 8 ? 64.0f : 1.0f;
    return fmaf(Act<TA>::to_f((uint16_t)s16) * up, (float)code * (1.0f / up), Act<TA>::to_f((uint16_t)b16));
}
// no number, or rounded past the type's largest?
template <typename TA>
__device__ __forceinline__ bool past_type(float v) {
    return !(fabsf(v) < (std::is_same<TA, __half>::value ? 65520.0f : 3.39617752923046e38f));
}
// Is a value of the group?  The values lie between the bias (code 0) and the
// last code's, and where the bias is no number the last is none either.
template <typename TA, int BITS>
__device__ __forceinline__ bool group_past_type(uint32_t s16, uint32_t b16) {
    return past_type<TA>(code_value<TA, BITS>((1u << BITS) - 1u, s16, b16));
}

int attn_num_sms();
// lmoe_attn.cu: joins the cut tiles of R rows of a launch of `grid` blocks; y: merge blocks for each
cudaError_t launch_attn_merge(int act_f16, int R, int D, int grid, int y, const AttnArgs &a, cudaStream_t st);
// lmoe_attn_chunk.cu
size_t chunk_scratch_bytes(int head_dim);
cudaError_t launch_attn_chunk(int act_f16, int head_dim, int bits, int group_size, const AttnArgs &a, cudaStream_t st);

}  // namespace lmoe
