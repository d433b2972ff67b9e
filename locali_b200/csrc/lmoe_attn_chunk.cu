// Attention of chunks (many rows of a sequence) over the paged key/value
// cache, on the 5th-generation tensor cores.
//
// A tile is 256 rows (tokens x query heads of one key/value head) as two
// sub-tiles of 128, the M of a tcgen05.mma; its keys are walked in blocks of
// 128 positions.  Per block and sub-tile t:
//   S_t = Q_t K^T            (Q_t, K in shared memory; S_t in tensor memory)
//   P_t = exp2(S_t c - m_t)  (one thread per row; P_t over S_t, in 16 bits)
//   O_t += P_t V             (P_t from tensor memory, V in shared memory)
// One block per SM; the stream of (tile, head, key block) is cut evenly over
// the launch as in lmoe_attn.cu.  Warp roles:
//   0-3, 4-7   softmax and output of sub-tile 0 and 1
//   8-11       keys into shared memory, 12-15 values: 16-bit rows by cp.async,
//              codes through registers, dequantised to the 16-bit type on the
//              way, into the 128-byte-swizzled operand layout
//   16, 17     one thread each issues the MMAs of sub-tile 0, 1
//   18         walks the launch block's tiles and lays what the others need to
//              know of them into a ring in shared memory
//   19         looks up the pages of the next key blocks for the loaders
// Register budgets differ (setmaxnreg): a softmax thread holds the 64 packed
// terms of its row.  ptxas still reports 650 to 680 bytes of spill stores in
// every instance, at the launch's 96 registers; 0.35 % of the instructions
// executed are local loads and stores (whole prompt of 4096, 16 bits).
// The sub-tiles issue their MMAs (P V of a block, then S of the next) in turn,
// which keeps them half a block apart: one's softmax overlaps the other's
// MMAs.  Issued as they came, the MMAs of both interleaved and ended together,
// and the two softmaxes then shared the exponential unit while the tensor pipe
// waited.  The reference of a row (Term in lmoe_attn.cuh) moves only when a score passes it
// by some powers of two: until then terms grow, which costs nothing in fp32
// and leaves the sums in tensor memory untouched.
//
// V is the MN-major B operand (head dimension contiguous), so keys and values
// share one layout: [D / 64][128 positions][128 bytes], 16-byte chunk c of
// position r at c ^ (r & 7).
//
// The floor is the tensor pipe (4 D flops per row and key; 2048 cycles a block
// at a head of 128) and beside it the exponentials (one per row and key, 16 a
// cycle: 2048 cycles too).  Measured on a B200: 2048 new tokens over 32 k
// cached, 32 query heads on 8, 8-bit codes: 1.15 ms a call behind an idle GPU
// (905 TFLOP/s, about 4400 cycles a block), 1.26 ms back to back.  What bounds
// it is the chain of one sub-tile: its softmax (about 2000 cycles, one thread a
// row), then P V and the next S (1100), then the hand-overs; without the
// softmax the same launch takes 0.72 ms, without dequantisation or its stores
// no less than with them.
#include "lmoe_attn.cuh"
#include "lmoe_tc.cuh"

namespace lmoe {

namespace {

constexpr int kCkRows = 256, kCkKeys = 128, kCkSub = 128;
constexpr int kCkThreads = 20 * 32;
constexpr int kCkLoadWarp = 8, kCkMmaWarp = 16, kCkWalkWarp = 18, kCkLookWarp = 19;
// Registers a thread after the split: 256 x 136 + 256 x 80 + 128 x 48 = 61440, the 640 x 96 of the launch.
constexpr int kRegSoftmax = 136, kRegLoad = 80, kRegRest = 48;
static_assert(256 * kRegSoftmax + 256 * kRegLoad + 128 * kRegRest <= kCkThreads * 96, "registers");
constexpr int kLook = 4;  // key blocks looked up ahead
constexpr int kSegs = 16;  // tiles in the ring: the look-up is at most 7 blocks ahead of the output
constexpr int kCkMinBlocks = 2;  // key blocks a launch block takes at least
constexpr int kCkTile = 4;       // what a tile costs besides its key blocks, in key blocks: its first block's extra
                                 // pass, its result and the hand-over are about 12k cycles, a block 3k
// Output staging of a warp: 32 rows of 64 bytes, 80 apart (no bank conflicts).  A lane holds a whole row, and rows
// stored straight from lanes touch 32 lines an instruction (an epilogue took 10k cycles).
constexpr int kStgRow = 80, kStgWarp = 32 * kStgRow;
constexpr int kExpFma = 2;  // of 8 pairs of exponentials, on the FMA pipe
constexpr int kPoison = 12;      // key blocks of a tile that some of its rows see in part: at most 8

// Keys of 64 elements dequantised to bf16 bring a second operand tile with
// what the rounding took off: rounded, they were most of a result's error (4.9e-3
// of its norm; the result's own rounding is 1.7e-3), and at 64 the tensor pipe
// and shared memory have room for it.  (At 128 they have not; f16 has three more
// bits.)
template <typename TA, int BITS, int D, int GS>
struct ChunkGeo {
    static constexpr bool LO = BITS != 16 && D == 64 && std::is_same<TA, __nv_bfloat16>::value;
    static constexpr int TILE = 128 * D * 2;  // an operand tile: 128 rows of D
    static constexpr int NG = BITS == 16 ? 1 : D / GS;
    static constexpr int OFF_Q = 0, OFF_K = 2 * TILE, OFF_V = 4 * TILE, OFF_L = 6 * TILE,
                         OFF_X = OFF_L + (LO ? 2 * TILE : 0);
    static constexpr int SCALES = BITS == 16 ? 0 : 8 * 32 * NG * (int)sizeof(uint2);  // scales and biases of the loader warps' rows
    static constexpr int OFF_STG = OFF_X + SCALES;                   // output staging of the softmax warps
    static constexpr int SMEM = 1024 + OFF_STG + 8 * kStgWarp;
};

// A tile, and the blocks of it that are this launch block's.
struct Seg {
    Tile t;
    int b0, b1;
    int more;   // another one follows
    int parts;  // launch blocks that share the tile, if it begins here and goes on behind; else 0
};

// A key block as the loaders need it: the head row where each 16-position run
// begins (-2: none, or none that a row sees, -1: no page).
struct Look {
    long long run[kCkKeys / 16];
    int left;  // positions in front of the end
    int blk, seg;
    int part;  // its number among the tile's blocks seen in part; -1: seen in full, -2: no block, the walk is over
};

// every row of the tile sees every position of the block at k0
__device__ __forceinline__ bool block_full(const AttnArgs &a, int k0, int minpos, int maxpos) {
    return k0 + kCkKeys - 1 <= minpos &&
           (a.window == 0 || k0 > (long long)maxpos - a.window || k0 + kCkKeys <= a.sinks);
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// the registers pass through, so no use of them moves above the wait
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// Shared-memory descriptor of an MN-major operand, 128-byte swizzle: 64
// elements of MN by 8 of K are one 1024-byte atom, the next 8 of K 1024 bytes
// on, the next 64 of MN 16 KB on.
__device__ __forceinline__ uint64_t mn128_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
// fp32 accumulator, M = 128, N = n, A K-major, B K-major or MN-major
__device__ __forceinline__ uint32_t attn_idesc(int n, bool f16, bool b_mn) {
    const uint32_t fmt = f16 ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}

// true in one lane of the converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(e));
    return e != 0;
}

// bits of [lo, hi) in the 32 positions from kb
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int kb) {
    const int l = min(max(lo - kb, 0), 32), h = min(max(hi - kb, 0), 32);
    return h > l ? (0xFFFFFFFFu >> (32 - (h - l))) << l : 0u;
}

// byte offset of 16-byte chunk c of row r in an operand tile
__device__ __forceinline__ uint32_t op_off(int r, int c) {
    return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename TA>
__device__ __forceinline__ bool nonfinite2(uint32_t x) {
    return nonfinite16<TA>(x) || nonfinite16<TA>(x >> 16);
}
// the pair with what is no number as zero
template <typename TA>
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
    if (nonfinite16<TA>(x)) x &= 0xFFFF0000u;
    if (nonfinite16<TA>(x >> 16)) x &= 0xFFFFu;
    return x;
}

// 8 codes -> 8 values as 16-bit pairs in order
template <typename TA, int BITS>
__device__ __forceinline__ uint4 dequant8(uint32_t w0, uint32_t w1, uint32_t s2, uint32_t b2) {
    uint32_t v[4];
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = Pair<TA>::value8(__byte_perm(i < 2 ? w0 : w1, 0u, i & 1 ? 0x4342 : 0x4140), s2, b2);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // codes 2i, 2i + 1 are the low nibbles of bytes i of the word and of it shifted
            v[i] = Pair<TA>::value4(__byte_perm(w0, w0 >> 4, i | (4 + i) << 8), 0, s2, b2);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// 2^x of a pair on the FMA pipe, for x up to 120 or so: x = n + f with n the
// nearest integer, 2^f by a polynomial on [-1/2, 1/2] (the minimax one of
// degree 4 with value 1 at 0, relative error 2.9e-6 in fp32), n added to the
// exponent.  Below -127 the result is 0.  An SM has 16 exponentials a cycle,
// half of what the tensor cores would have of a row's scores at a head of 128.
__device__ __forceinline__ void exp2_fma(float &x, float &y) {
    const uint64_t magic = pack_f2(12582912.0f, 12582912.0f), unmagic = pack_f2(-12582912.0f, -12582912.0f);
    const uint64_t v = pack_f2(fmaxf(x, -127.0f), fmaxf(y, -127.0f));
    const uint64_t t = add_f2(v, magic);  // n in the low bits
    const uint64_t f = fma_f2(add_f2(t, unmagic), pack_f2(-1.0f, -1.0f), v);
    uint64_t p = pack_f2(0.009582852944731712f, 0.009582852944731712f);
    p = fma_f2(p, f, pack_f2(0.055906426161527634f, 0.055906426161527634f));
    p = fma_f2(p, f, pack_f2(0.24024099111557007f, 0.24024099111557007f));
    p = fma_f2(p, f, pack_f2(0.6931241750717163f, 0.6931241750717163f));
    p = fma_f2(p, f, pack_f2(1.0f, 1.0f));
    float p0, p1, t0, t1;
    unpack_f2(p, p0, p1);
    unpack_f2(t, t0, t1);
    x = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
    y = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}
// largest of three, keeping a NaN
__device__ __forceinline__ float max3_nan(float x, float y, float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// tcgen05.ld and st of one column
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r)
                 : "r"(taddr)
                 : "memory");
    return __uint_as_float(r);
}
__device__ __forceinline__ void tmem_st1(uint32_t taddr, float v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(taddr),
                 "r"(__float_as_uint(v))
                 : "memory");
}

// Largest visible score of the thread's row, S at `ts`; mask(c) has the bits
// of columns 32 c .. 32 c + 31.  Not unrolled: it runs for a tile's first
// block and for blocks seen in part, and unrolled code that runs so seldom is
// fetched anew each time.
template <class F>
__device__ __forceinline__ float row_max(uint32_t ts, F &&mask, bool &seen) {
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        const uint32_t mk = mask(c);
        if (!__any_sync(0xffffffffu, mk != 0)) continue;
        seen |= mk != 0;
        uint32_t v[32];
        tmem_ld32(ts + 32 * c, v);
        tmem_wait_ld32(v);
        if (!__all_sync(0xffffffffu, mk == 0xFFFFFFFFu)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (!(mk >> e & 1u)) v[e] = 0xFF800000u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            x0 = max3_nan(x0, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            x1 = max3_nan(x1, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
        }
    }
    return max_nan(x0, x1);
}

// Terms exp2(S sc - mu) over S, as 16-bit pairs for the tensor core (32
// columns of S become 16, behind the reads); returns their sum in fp32.
template <typename TA, class F>
__device__ __forceinline__ float row_terms(uint32_t ts, F &&mask, float sc, float mu) {
    const uint64_t sc2 = pack_f2(sc, sc), mu2 = pack_f2(-mu, -mu);
    uint64_t sum = 0;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        const uint32_t mk = mask(c);
        uint32_t pk[16];
        if (!__any_sync(0xffffffffu, mk != 0)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] = 0u;
        } else {
            uint32_t v[32];
            tmem_ld32(ts + 32 * c, v);
            tmem_wait_ld32(v);
            if (!__all_sync(0xffffffffu, mk == 0xFFFFFFFFu)) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (!(mk >> e & 1u)) v[e] = 0xFF800000u;  // sc > 0: its term is 0
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                float p0, p1;
                unpack_f2(fma_f2(pack_f2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc2, mu2), p0, p1);
                p0 = ex2(p0);
                p1 = ex2(p1);
                sum = add_f2(sum, pack_f2(p0, p1));
                pk[e / 2] = Act<TA>::pack2(p0, p1);
            }
        }
        tmem_st16(ts + 16 * c, pk);
    }
    float s0, s1;
    unpack_f2(sum, s0, s1);
    return s0 + s1;
}

// Terms over an S seen in full with the reference m as it is, in one read;
// nothing is written (again = true) when a term of a row of the warp passes
// the largest there may be or a score is no number.
template <typename TA>
__device__ __forceinline__ float row_try(uint32_t ts, float sc, float m, bool &again) {
    const float mu = m == -INFINITY ? 0.0f : m;
    const uint64_t sc2 = pack_f2(sc, sc), mu2 = pack_f2(-mu, -mu);
    uint64_t sum = 0;
    float x0 = -INFINITY, x1 = -INFINITY;
    uint32_t pk[64];
    auto take = [&](uint32_t (&v)[16], int c) {  // columns 16 c ..
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            x0 = max3_nan(x0, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            x1 = max3_nan(x1, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            float p0, p1;
            unpack_f2(fma_f2(pack_f2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc2, mu2), p0, p1);
            if (e / 2 % 8 < kExpFma) {
                exp2_fma(p0, p1);
            } else {
                p0 = ex2(p0);
                p1 = ex2(p1);
            }
            sum = add_f2(sum, pack_f2(p0, p1));
            pk[8 * c + e / 2] = Act<TA>::pack2(p0, p1);
        }
    };
    uint32_t v[16], y[16];
    tmem_ld16(ts, v);
    tmem_wait_ld(v);
#pragma unroll
    for (int c = 0; c < 8; c += 2) {
        tmem_ld16(ts + 16 * (c + 1), y);
        take(v, c);
        tmem_wait_ld(y);
        if (c < 6) tmem_ld16(ts + 16 * (c + 2), v);
        take(y, c + 1);
        if (c < 6) tmem_wait_ld(v);
    }
    const float x = max_nan(x0, x1) * sc;
    again = __any_sync(0xffffffffu, !(x <= m + Term<TA, true>::kTop) && !(x == -INFINITY));
    if (!again) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t z[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) z[e] = pk[32 * h + e];
            tmem_st32(ts + 32 * h, z);
        }
    }
    float s0, s1;
    unpack_f2(sum, s0, s1);
    return s0 + s1;
}

// What rounding scale * code + bias to the 8 bf16 values v took off them
// (s2 as dequant8 takes it).
template <int BITS>
__device__ __forceinline__ uint4 dequant8_rest(uint32_t w0, uint32_t w1, uint32_t s2, uint32_t b2, const uint4 &v) {
    const float s = __uint_as_float(s2 << 16) * (BITS == 8 ? 1.0f / 64.0f : 1.0f), b = __uint_as_float(b2 << 16);
    const uint32_t hi[4] = {v.x, v.y, v.z, v.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = BITS == 8 ? (i < 2 ? w0 : w1) >> (16 * (i & 1)) : w0 >> (8 * i);
        const uint32_t c0 = w & (BITS == 8 ? 255u : 15u), c1 = w >> BITS & (BITS == 8 ? 255u : 15u);
        // 2^23 + code as a number
        const float f0 = __uint_as_float(0x4B000000u | c0) - 8388608.0f, f1 = __uint_as_float(0x4B000000u | c1) - 8388608.0f;
        r[i] = Act<__nv_bfloat16>::pack2(fmaf(s, f0, b) - __uint_as_float(hi[i] << 16),
                                         fmaf(s, f1, b) - __uint_as_float(hi[i] & 0xFFFF0000u));
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename TA, int BITS, int D, int GS>
__global__ void __launch_bounds__(kCkThreads, 1) attn_chunk_kernel(const AttnArgs a) {
    using G = ChunkGeo<TA, BITS, D, GS>;
    constexpr int CH = D / 8;   // 16-byte chunks of an operand row
    constexpr int RB = D * BITS / 8;
    constexpr bool Q = BITS != 16;
    constexpr int NG = G::NG;
    constexpr bool F16 = std::is_same<TA, __half>::value;
    extern __shared__ __align__(1024) uint8_t raw[];
    __shared__ long long s_plan[kCkThreads / 32 + 4];
    __shared__ uint32_t s_bad[8];  // block u & 7: its runs without a page
    __shared__ uint32_t s_poison[4][kPoison][4];  // tile & 3, its n-th block seen in part: rows taken out
    __shared__ int s_pblk[4][kPoison];
    __shared__ Look s_look[kLook];
    __shared__ uint64_t bars[18 + 2 * kSegs + 2 * kLook];
    __shared__ Seg s_seg[kSegs];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    uint8_t *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6, *sfull = bars + 8,
             *pfull = bars + 10, *qfull = bars + 12, *ofull = bars + 14, *turn = bars + 16,
             *gfull = bars + 18, *gempty = gfull + kSegs, *lfull = gempty + kSegs, *lempty = lfull + kLook;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&kfull[i], 4);
            mbar_init(&kempty[i], 2);
            mbar_init(&vfull[i], 4);
            mbar_init(&vempty[i], 2);
            mbar_init(&sfull[i], 1);
            mbar_init(&pfull[i], 4);
            mbar_init(&qfull[i], 4);
            mbar_init(&ofull[i], 1);
            mbar_init(&turn[i], 1);
        }
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(&gfull[i], 1);
            mbar_init(&gempty[i], 11);  // 8 softmax warps, 2 MMA warps, the look-up
        }
        for (int i = 0; i < kLook; ++i) {
            mbar_init(&lfull[i], 1);
            mbar_init(&lempty[i], 8);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0) a.r.validate(threadIdx.x, kCkThreads);
    MergeRec *rec = reinterpret_cast<MergeRec *>(a.scratch) + blockIdx.x;
    if (threadIdx.x == 0) rec->parts = 0;
    Share sh;
    Cursor<kCkRows, kCkKeys, kCkTile> cur;
    const bool work =
        a.r.n_seqs <= 2 * (kCkThreads / 32)
            ? find_share<kCkRows, kCkKeys, kCkTile, kCkThreads, true>(a, kCkTile + kCkMinBlocks, s_plan, sh, cur)
            : find_share<kCkRows, kCkKeys, kCkTile, kCkThreads, false>(a, kCkTile + kCkMinBlocks, s_plan, sh, cur);
    if (!work) return;
    if (warp == kCkMmaWarp) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    // tensor memory columns: S_0 (P_0), S_1 (P_1), O_0, O_1
    auto tm_s = [&](int t) { return tmem + (uint32_t)(t * 128); };
    auto tm_o = [&](int t) { return tmem + (uint32_t)(256 + t * D); };

    // a wait that gave up: the error is latched and every role leaves
    auto wait = [&](uint64_t *bar, uint32_t ph) -> bool {
        if (pf_wait(bar, ph)) return true;
        s_abort = 1;
        set_error(a.r.err, kErrCuda);
        return false;
    };
    // the launch block's n-th tile; let go (by one lane of each warp) when nothing more of it is needed
    auto seg = [&](int n) -> const Seg & { return s_seg[n % kSegs]; };
    auto seg_ready = [&](int n) -> bool { return wait(&gfull[n % kSegs], n / kSegs & 1); };
    auto seg_done = [&](int n) { mbar_arrive(&gempty[n % kSegs]); };

    if (warp < kCkLoadWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegSoftmax));
        // ---------------------------------------------------- softmax and output
        const int t = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane;  // row of the sub-tile
        const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
        const uint32_t qs = sb + G::OFF_Q + t * G::TILE;
        const float sc = a.scale_log2;
        // the row's query into the operand tile (zeros where there is none)
        auto load_q = [&](const Tile &ti) {
            const int row = ti.rt * kCkRows + t * kCkSub + r;
            const bool in = row < ti.n * a.group;
            const int tok = in ? a.per_group(row) : 0;
            const uint16_t *src = a.q + (int64_t)(ti.row0 + tok) * a.q_tok_stride +
                                  (int64_t)(ti.h * a.group + (in ? row - tok * a.group : 0)) * a.q_head_stride;
            // CH lanes a row, 32 / CH rows at a time
            const uint32_t ins = __ballot_sync(0xffffffffu, in);
            const int cc = lane % CH;
#pragma unroll 4
            for (int x = lane / CH; x < 32; x += 32 / CH) {
                const uint16_t *p = reinterpret_cast<const uint16_t *>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), x));
                const bool ok = ins >> x & 1u;
                cp16z(qs + op_off(q4 * 32 + x, cc), ok ? p + cc * 8 : a.q, ok ? 16 : 0);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int u = 0, act = 0, active_segs = 0;
        bool ok = __all_sync(0xffffffffu, seg_ready(0));
        if (ok) load_q(seg(0).t);
        for (int n = 0; ok && !s_abort; ++n) {
            const Seg &sg = seg(n);
            const Tile &ti = sg.t;
            const int b0 = sg.b0, b1 = sg.b1, more = sg.more;
            if (t == 1 && ti.rows <= kCkSub) {
                // no rows: only pass the tiles of keys and values on
                if (r == 0)
                    for (int i = b0; i < b1 && ok; ++i) {
                        const int s = (u + i - b0) & 1, ph = (u + i - b0) >> 1 & 1;
                        ok = wait(&kfull[s], ph);
                        if (ok) mbar_arrive(&kempty[s]);
                        ok = ok && wait(&vfull[s], ph);
                        if (ok) mbar_arrive(&vempty[s]);
                    }
                u += b1 - b0;
                ok = __all_sync(0xffffffffu, ok && (!more || seg_ready(n + 1)));
                asm volatile("cp.async.wait_group 0;" ::: "memory");  // before the same rows are written again
                if (ok && more) load_q(seg(n + 1).t);
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&qfull[t]);
                const int row = ti.rt * kCkRows + t * kCkSub + r;
                const bool in = row < ti.n * a.group;
                const int p = in ? ti.first + a.per_group(row) : -1;
                const int see_hi = min(p + 1, ti.hi), see_lo = a.window ? (int)max(0ll, (long long)p - a.window + 1) : 0;
                const int see_sink = min(a.sinks, see_hi);
                // positions of the sub-tile's first and last row
                const int lastrow = min(ti.rows, (t + 1) * kCkSub) - 1;
                const int nsink = ti.nsink, lo = ti.lo - nsink;
                const int tmin = min(ti.minpos, ti.hi - 1), tmax = ti.maxpos;
                const int smin = min(ti.first + a.per_group(ti.rt * kCkRows + t * kCkSub), ti.hi - 1);
                const int smax = ti.first + a.per_group(ti.rt * kCkRows + lastrow);
                float m = -INFINITY;
                float l = 0.0f;
                bool seen = false;
                int parts = 0;
                for (int i = b0; i < b1; ++i, ++u, ++act) {
                    const int k0 = (i < nsink ? i : lo + i) * kCkKeys;
                    ok = __all_sync(0xffffffffu, wait(&sfull[t], act & 1));
                    if (!ok) break;
                    tc_fence_after();
                    if (r == 0) {  // the MMAs before S_t's end are done: the keys, and the values before
                        mbar_arrive(&kempty[u & 1]);
                        if (i > b0) mbar_arrive(&vempty[(u - 1) & 1]);
                    }
                    const uint32_t bad = s_bad[u & 7];
                    const bool full = !bad && block_full(a, k0, smin, smax);
                    if (!block_full(a, k0, tmin, tmax)) ++parts;
                    auto mask = [&](int c) -> uint32_t {
                        if (full) return 0xFFFFFFFFu;
                        const int kb = k0 + 32 * c;
                        uint32_t x = range_bits(see_lo, see_hi, kb) | range_bits(0, see_sink, kb);
                        if (bad >> (2 * c) & 1u) x &= 0xFFFF0000u;
                        if (bad >> (2 * c) & 2u) x &= 0x0000FFFFu;
                        return x;
                    };
                    // with the reference as it is, unless a score of the block passes it
                    const uint32_t ts = tm_s(t) + lanes;
                    bool again = true;
                    if (full && i > b0) {
                        seen = true;
                        const float sum = row_try<TA>(ts, sc, m, again);
                        if (!again) l += sum;
                    }
                    if (again) {
                        const float x = row_max(ts, mask, seen) * sc;
                        const bool move = !(x <= m + Term<TA, true>::kTop) && !(x == -INFINITY);
                        if (__any_sync(0xffffffffu, move)) {
                            const float to = x - Term<TA, true>::kSet, f = move ? ex2(m - to) : 1.0f;
                            if (move) m = to;
                            l *= f;
                            if (i > b0) {  // the sums so far
#pragma unroll 1
                                for (int c = 0; c < D / 32; ++c) {
                                    uint32_t v[32];
                                    tmem_ld32(tm_o(t) + lanes + 32 * c, v);
                                    tmem_wait_ld32(v);
#pragma unroll
                                    for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                                    tmem_st32(tm_o(t) + lanes + 32 * c, v);
                                }
                            }
                        }
                        l += row_terms<TA>(ts, mask, sc, m == -INFINITY ? 0.0f : m);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pfull[t]);
                }
                if (!ok) break;
                if (more) {  // Q_t is free
                    ok = __all_sync(0xffffffffu, seg_ready(n + 1));
                    if (!ok) break;
                    load_q(seg(n + 1).t);
                }
                // ---- the tile's result
                ok = __all_sync(0xffffffffu, wait(&ofull[t], active_segs & 1));
                ++active_segs;
                if (!ok) break;
                tc_fence_after();
                if (r == 0) mbar_arrive(&vempty[(u - 1) & 1]);
                // only scores of -inf: the softmax is no number, unless other
                // parts of the tile's keys hold larger ones
                if (m == -INFINITY && seen) l = __uint_as_float(0x7FC00000u);
                const bool whole = b0 == 0 && b1 == ti.nblk;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                bool poisoned = false;
                for (int pi = 0; pi < parts; ++pi)
                    poisoned |= (s_poison[n & 3][pi][0] | s_poison[n & 3][pi][1] | s_poison[n & 3][pi][2] | s_poison[n & 3][pi][3]) != 0;
                if (poisoned) {
                    // values that are no numbers, taken out of blocks that
                    // only some rows see: added for those that do
#pragma unroll 1
                    for (int x = 0; x < parts * kCkKeys; ++x) {
                        const int pi = x / kCkKeys, k = x % kCkKeys;
                        if (!(s_poison[n & 3][pi][k >> 5] >> (k & 31) & 1u)) continue;
                        const int j = s_pblk[n & 3][pi] * kCkKeys + k;
                        const bool sees = j < see_hi && (j >= see_lo || j < see_sink);
                        const int32_t pg = a.r.page(a.c, ti.b, j);
                        if (pg < 0) continue;
                        const int64_t kr = a.c.row(pg, ti.h, a.c.slot_of(j));
#pragma unroll 1
                        for (int d = 0; d < D; ++d) {
                            float y;
                            if constexpr (Q) {
                                const uint32_t by = a.c.kv[1][kr * RB + d * BITS / 8];
                                const uint32_t code = BITS == 8 ? by : by >> (4 * (d & 1)) & 15u;
                                y = code_value<TA, BITS>(code, a.c.scale[1][kr * NG + d / GS], a.c.bias[1][kr * NG + d / GS]);
                            } else {
                                y = Act<TA>::to_f(reinterpret_cast<const uint16_t *>(a.c.kv[1])[kr * D + d]);
                            }
                            if (!past_type<TA>(y)) continue;  // the same for all lanes
                            y *= INFINITY;
                            const float o = tmem_ld1(tm_o(t) + lanes + d);
                            tmem_st1(tm_o(t) + lanes + d, sees ? o + y : o);
                        }
                    }
                }
                // rows go out through the staging, 4 lanes a row of 64 bytes
                const uint32_t stg = sb + G::OFF_STG + warp * kStgWarp;
                const int tok = in ? a.per_group(row) : 0;
                uint8_t *to = whole ? reinterpret_cast<uint8_t *>(a.out + ((int64_t)ti.row0 * a.q_heads + ti.h * a.group) * D)
                                    : reinterpret_cast<uint8_t *>(part_ptr(a, gridDim.x, part_floats<kCkRows, D>(),
                                                                           blockIdx.x, b0 == 0 ? 1 : 0));
                // the row's offset, 64 bytes at a time: it fits 32 bits for results of up to 2^38 bytes (kMaxOut)
                const uint32_t mine = whole ? (uint32_t)(((int64_t)tok * (a.q_heads - a.group) + row) * (D * 2 / 64))
                                            : (uint32_t)((t * kCkSub + r) * (D * 4 / 64));
                uint8_t *dst[4];
                const uint32_t ins = __ballot_sync(0xffffffffu, in);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    dst[x] = to + (int64_t)__shfl_sync(0xffffffffu, mine, 8 * x + (lane >> 2)) * 64 + (lane & 3) * 16;
                const int cols = whole ? 32 : 16;  // columns of 64 bytes
#pragma unroll 1
                for (int c = 0; c < D; c += cols) {
                    uint4 o[4];
                    uint32_t *ov = &o[0].x;
                    if (whole) {
                        uint32_t v[32];
                        tmem_ld32(tm_o(t) + lanes + c, v);
                        tmem_wait_ld32(v);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            ov[e] = Act<TA>::pack2(__uint_as_float(v[2 * e]) * inv, __uint_as_float(v[2 * e + 1]) * inv);
                    } else {
                        uint32_t v[16];
                        tmem_ld16(tm_o(t) + lanes + c, v);
                        tmem_wait_ld(v);
#pragma unroll
                        for (int e = 0; e < 16; ++e) ov[e] = v[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) sts128v(stg + lane * kStgRow + e * 16, o[e].x, o[e].y, o[e].z, o[e].w);
                    __syncwarp();
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint4 v = lds128(stg + (8 * x + (lane >> 2)) * kStgRow + (lane & 3) * 16);
                        if (ins >> (8 * x + (lane >> 2)) & 1u) *reinterpret_cast<uint4 *>(dst[x]) = v;
                        dst[x] += 64;
                    }
                    __syncwarp();
                }
                if (!whole) {
                    float2 *ml = reinterpret_cast<float2 *>(
                        part_ptr(a, gridDim.x, part_floats<kCkRows, D>(), blockIdx.x, b0 == 0 ? 1 : 0) + kCkRows * D);
                    ml[t * kCkSub + r] = make_float2(m, l);
                }
                if (t == 0 && r == 0 && sg.parts) {
                    rec->out0 = ti.row0;
                    rec->row = ti.rt * kCkRows;
                    rec->rows_h = ti.rows | ti.h << 16;
                    rec->parts = sg.parts;
                }
                // O_t is read: the next tile's first P_t says so
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) seg_done(n);
            if (!more) break;
        }
    } else if (warp < kCkMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegLoad));
        // ---------------------------------------------------- keys and values
        const int which = (warp - kCkLoadWarp) >> 2, lw = warp & 3;  // rows 32 lw .. of a block
        uint64_t *fullb = which ? vfull : kfull, *emptyb = which ? vempty : kempty;
        const uint8_t *const kv = a.c.kv[which];
        const uint32_t base = sb + (which ? G::OFF_V : G::OFF_K);
        constexpr int LPR = CH, RPI = 32 / LPR, IT = 32 / RPI;  // lanes of a row; rows and rounds of a warp's 32
        const int rr = lane / LPR, cc = lane % LPR;
        const int64_t lane_off = (int64_t)rr * RB + cc * BITS;  // the lane's part of a round's rows
        // the warp's share of a block
        struct Unit {
            long long r0, r1;  // head rows of its two runs
            int left, blk, seg, part;
        };
        auto look = [&](int u) -> Unit {
            Unit n{-2, -2, 0, 0, 0, -2};
            if (!__all_sync(0xffffffffu, wait(&lfull[u % kLook], u / kLook & 1))) return n;
            const Look &e = s_look[u % kLook];
            n = Unit{e.run[2 * lw], e.run[2 * lw + 1], e.left - 32 * lw, e.blk, e.seg, e.part};
            __syncwarp();
            if (lane == 0) mbar_arrive(&lempty[u % kLook]);
            return n;
        };
        // head row of the warp's row x, -1 where there is nothing to read
        auto row_of = [&](const Unit &n, int x) -> long long {
            const long long r = x < 16 ? n.r0 : n.r1;
            return r >= 0 && x < n.left ? r + (x & 15) : -1;
        };
        auto whole = [&](const Unit &n) { return n.r0 >= 0 && n.r1 >= 0 && n.left >= 32; };
        auto empty = [&](int u) -> bool { return __all_sync(0xffffffffu, wait(&emptyb[u & 1], (u >> 1 & 1) ^ 1)); };
        // the share is in place; taken: its rows with values taken out
        auto done = [&](const Unit &n, int u, uint32_t taken) {
            if (which && n.part >= 0 && lane == 0) {
                s_poison[n.seg & 3][n.part][lw] = taken;
                if (lw == 0) s_pblk[n.seg & 3][n.part] = n.blk;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&fullb[u & 1]);
        };
        if constexpr (Q) {
            constexpr int WPC = BITS == 8 ? 2 : 1;  // code words of a chunk
            uint32_t code[IT][WPC];
            uint32_t sc[(NG + 1) / 2], bi[(NG + 1) / 2];  // of row `lane`, two groups a word
            bool in_lane = false;                        // row `lane` is there
            // (scale, scale), (bias, bias) of the rows' groups
            uint2 *spair = reinterpret_cast<uint2 *>(smem + G::OFF_X) + (warp - kCkLoadWarp) * 32 * NG;
            // all loads of a share, issued as soon as the one before it is in place
            auto fetch = [&](const Unit &n) {
                const long long r = row_of(n, lane);
                const uint16_t *ps = a.c.scale[which] + (r < 0 ? 0 : r * NG), *pb = a.c.bias[which] + (r < 0 ? 0 : r * NG);
                if constexpr (NG == 1) {
                    sc[0] = *ps;
                    bi[0] = *pb;
                } else if constexpr (NG == 2) {
                    sc[0] = *reinterpret_cast<const uint32_t *>(ps);
                    bi[0] = *reinterpret_cast<const uint32_t *>(pb);
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(ps), y = *reinterpret_cast<const uint2 *>(pb);
                    sc[0] = x.x;
                    sc[(NG - 1) / 2] = x.y;
                    bi[0] = y.x;
                    bi[(NG - 1) / 2] = y.y;
                }
                in_lane = r >= 0;
                const uint8_t *p0 = kv + lane_off + n.r0 * RB, *p1 = kv + lane_off + n.r1 * RB;
                auto get = [&](int x, bool in) {
                    const uint8_t *src = (x * RPI < 16 ? p0 : p1) + (x * RPI % 16) * RB;
                    if constexpr (BITS == 8) {
                        const uint2 v = in ? *reinterpret_cast<const uint2 *>(src) : make_uint2(0u, 0u);
                        code[x][0] = v.x;
                        code[x][1] = v.y;
                    } else {
                        code[x][0] = in ? *reinterpret_cast<const uint32_t *>(src) : 0u;
                    }
                };
                if (whole(n)) {
#pragma unroll
                    for (int x = 0; x < IT; ++x) get(x, true);
                } else {
#pragma unroll
                    for (int x = 0; x < IT; ++x) get(x, row_of(n, x * RPI + rr) >= 0);
                }
            };
            // the share into its place, four rounds at a time so that their reads and arithmetic overlap
            auto put = [&](const Unit &n, int u) {
                bool no = false;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t x = in_lane ? __byte_perm(sc[g / 2], bi[g / 2], g & 1 ? 0x7632 : 0x5410) : 0u;
                    // in a block that only some rows see, values that are no numbers are taken out
                    if (which && n.part >= 0) no |= group_past_type<TA, BITS>(x & 0xFFFFu, x >> 16);
                    spair[lane * NG + g] = make_uint2(Pair<TA>::template scale<BITS>(__byte_perm(x, 0u, 0x1010)),
                                                      __byte_perm(x, 0u, 0x3232));
                }
                const uint32_t taken = __ballot_sync(0xffffffffu, no);
                __syncwarp();
                const uint32_t dst = base + (u & 1) * G::TILE;
                const uint2 *sp = spair + rr * NG + cc * 8 / GS;
#pragma unroll
                for (int x0 = 0; x0 < IT; x0 += 4) {
                    uint2 sv[4];
                    uint4 v[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) sv[x] = sp[(x0 + x) * RPI * NG];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        v[x] = dequant8<TA, BITS>(code[x0 + x][0], code[x0 + x][WPC - 1], sv[x].x, sv[x].y);
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        sts128v(dst + op_off(lw * 32 + (x0 + x) * RPI + rr, cc), v[x].x, v[x].y, v[x].z, v[x].w);
                    if (G::LO && !which) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint4 y = dequant8_rest<BITS>(code[x0 + x][0], code[x0 + x][WPC - 1], sv[x].x, sv[x].y, v[x]);
                            sts128v(dst - G::OFF_K + G::OFF_L + op_off(lw * 32 + (x0 + x) * RPI + rr, cc), y.x, y.y, y.z, y.w);
                        }
                    }
                }
                if (taken) {  // the lane's own stores
#pragma unroll 1
                    for (int x = 0; x < IT; ++x) {
                        const uint32_t at = dst + op_off(lw * 32 + x * RPI + rr, cc);
                        const uint4 v = lds128(at);
                        sts128v(at, finite2<TA>(v.x), finite2<TA>(v.y), finite2<TA>(v.z), finite2<TA>(v.w));
                    }
                }
                done(n, u, taken);
            };
            Unit n = look(0);
            if (n.part > -2) fetch(n);
            for (int u = 0; n.part > -2 && !s_abort; ++u) {
                if (!empty(u)) break;
                put(n, u);
                n = look(u + 1);
                if (n.part > -2) fetch(n);
            }
        } else {
            auto copy = [&](const Unit &n, int u) {
                const uint32_t dst = base + (u & 1) * G::TILE;
                if (whole(n)) {
                    const uint8_t *p0 = kv + lane_off + n.r0 * RB, *p1 = kv + lane_off + n.r1 * RB;
#pragma unroll
                    for (int x = 0; x < IT; ++x)
                        cp16z(dst + op_off(lw * 32 + x * RPI + rr, cc), (x * RPI < 16 ? p0 : p1) + (x * RPI % 16) * RB, 16);
                } else {
#pragma unroll 1
                    for (int x = 0; x < IT; ++x) {
                        const long long r = row_of(n, x * RPI + rr);
                        cp16z(dst + op_off(lw * 32 + x * RPI + rr, cc), r >= 0 ? kv + r * RB + cc * 16 : kv, r >= 0 ? 16 : 0);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            // the copies of a share have landed
            auto finish = [&](const Unit &n, int u) {
                uint32_t taken = 0;
                if (which && n.part >= 0) {
                    __syncwarp();
#pragma unroll 1
                    for (int x = 0; x < IT; ++x) {
                        const uint32_t at = base + (u & 1) * G::TILE + op_off(lw * 32 + x * RPI + rr, cc);
                        uint4 v = lds128(at);
                        const bool no = nonfinite2<TA>(v.x) || nonfinite2<TA>(v.y) || nonfinite2<TA>(v.z) || nonfinite2<TA>(v.w);
                        const uint32_t bl = __ballot_sync(0xffffffffu, no);
                        if (bl == 0) continue;
                        if (no) sts128v(at, finite2<TA>(v.x), finite2<TA>(v.y), finite2<TA>(v.z), finite2<TA>(v.w));
#pragma unroll
                        for (int y = 0; y < RPI; ++y)
                            if (bl >> (y * LPR) & ((1u << LPR) - 1u)) taken |= 1u << (x * RPI + y);
                    }
                }
                done(n, u, taken);
            };
            // One share is in flight while the one before it is completed,
            // unless its place is still taken: then that one first.
            Unit prev{};
            bool pending = false, ok = true;
            int u = 0;
            for (; !s_abort; ++u) {
                const Unit n = look(u);
                if (n.part == -2) break;
                if (pending && !__all_sync(0xffffffffu, mbar_test(&emptyb[u & 1], (u >> 1 & 1) ^ 1))) {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    finish(prev, u - 1);
                    pending = false;
                }
                ok = empty(u);
                if (!ok) break;
                copy(n, u);
                if (pending) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    finish(prev, u - 1);
                }
                prev = n;
                pending = true;
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (pending && ok) finish(prev, u - 1);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegRest));
    }
    if (warp >= kCkMmaWarp && warp < kCkMmaWarp + 2) {
        // ---------------------------------------------------- MMAs of sub-tile t
        // The whole warp walks along and one elected lane issues: with the
        // control flow uniform, the descriptors stay in uniform registers.
        // (Issued from a lane's own branch, every MMA first moved its operands
        // there, and the issue took longer than the MMAs.)
        const int t = __shfl_sync(0xffffffffu, warp - kCkMmaWarp, 0);
        const uint32_t id_s = attn_idesc(kCkKeys, F16, false), id_o = attn_idesc(D, F16, true);
        const uint32_t sbu = __shfl_sync(0xffffffffu, sb, 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t ds = tm + (uint32_t)(t * 128), dd = tm + (uint32_t)(256 + t * D);
        const uint64_t qd = sw128_desc(sbu + G::OFF_Q + t * G::TILE);
        auto all = [&](bool x) -> bool { return __all_sync(0xffffffffu, x); };
        auto scores = [&](int u) {
            const uint64_t kd = sw128_desc(sbu + G::OFF_K + (u & 1) * G::TILE);
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    const uint64_t o = (uint64_t)((s >> 2) * (16384 >> 4) + (s & 3) * 2);
                    umma_f16(ds, qd + o, kd + o, id_s, s ? 1u : 0u);
                }
                if constexpr (G::LO) {
                    const uint64_t ld = sw128_desc(sbu + G::OFF_L + (u & 1) * G::TILE);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) umma_f16(ds, qd + s * 2, ld + s * 2, id_s, 1u);
                }
            }
            __syncwarp();
        };
        auto commit = [&](uint64_t *bar) {
            if (elect_one()) umma_commit(bar);
            __syncwarp();
        };
        int u = 0, act = 0, active_segs = 0;
        bool ok = true;
        for (int n = 0; !s_abort; ++n) {
            if (!all(seg_ready(n))) break;
            const int nb = __shfl_sync(0xffffffffu, seg(n).b1 - seg(n).b0, 0);
            const int rows = __shfl_sync(0xffffffffu, seg(n).t.rows, 0), more = __shfl_sync(0xffffffffu, seg(n).more, 0);
            if (lane == 0) seg_done(n);
            __syncwarp();
            if (t == 1 && rows <= kCkSub) {
                for (int j = 0; j < nb && ok; ++j, ++u) {  // only pass the turn on
                    ok = all(wait(&turn[1], u & 1));
                    if (ok && lane == 0) mbar_arrive(&turn[0]);
                    __syncwarp();
                }
            } else {
                ok = all(wait(&qfull[t], active_segs & 1) && wait(&kfull[u & 1], u >> 1 & 1));
                ++active_segs;
                if (!ok) break;
                tc_fence_after();
                scores(u);
                commit(&sfull[t]);
                for (int j = 0; j < nb; ++j, ++u, ++act) {
                    const bool last = j + 1 == nb;
                    ok = all(wait(&vfull[u & 1], u >> 1 & 1) && (last || wait(&kfull[(u + 1) & 1], (u + 1) >> 1 & 1)) &&
                             wait(&pfull[t], act & 1) && wait(&turn[t], t ? u & 1 : (u & 1) ^ 1));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = mn128_desc(sbu + G::OFF_V + (u & 1) * G::TILE);
                    if (elect_one()) {
#pragma unroll
                        for (int s = 0; s < kCkKeys / 16; ++s)
                            umma_f16_ts(dd, ds + 8 * s, vd + (uint64_t)(s * (2048 >> 4)), id_o, s ? 1u : (uint32_t)(j != 0));
                    }
                    __syncwarp();
                    if (!last) scores(u + 1);
                    if (lane == 0) mbar_arrive(&turn[t ^ 1]);
                    commit(last ? &ofull[t] : &sfull[t]);
                }
            }
            if (!ok || !more) break;
        }
    } else if (warp == kCkWalkWarp && lane == 0) {
        // ---------------------------------------------------- the walk
        bool more = true;
        for (int n = 0; more && !s_abort; ++n) {
            if (n >= kSegs && !wait(&gempty[n % kSegs], (n / kSegs - 1) & 1)) break;
            Seg &sg = s_seg[n % kSegs];
            sg.t = cur.t;
            sg.b0 = cur.b0;
            sg.b1 = cur.b1;
            sg.parts = cur.shared(sh, blockIdx.x);
            more = cur.next(a);
            sg.more = more;
            mbar_arrive(&gfull[n % kSegs]);
        }
    } else if (warp == kCkLookWarp) {
        // ---------------------------------------------------- the pages of the key blocks
        // lane x < 8: run x of the block; the page ids of a block are asked
        // for before those of the one in front of it are looked at
        int u = 0;
        Look e;  // the block asked for (run: not used)
        int32_t page = -1;
        int slot = -1, head = 0;
        e.part = -2;
        auto give = [&]() -> bool {
            if (u >= kLook && !__all_sync(0xffffffffu, wait(&lempty[u % kLook], (u / kLook - 1) & 1))) return false;
            long long run = -2;
            if (slot >= 0) {
                const bool in = page >= 0 && page < a.c.n_pages;
                if (!in) set_error(a.r.err, kErrIndex);
                run = in ? a.c.row(page, head, slot) : -1;
            }
            const uint32_t bad = __ballot_sync(0xffffffffu, run == -1);
            Look &x = s_look[u % kLook];
            if (lane < kCkKeys / 16) x.run[lane] = run;
            if (lane == 0) {
                x.left = e.left;
                x.blk = e.blk;
                x.seg = e.seg;
                x.part = e.part;
                s_bad[u & 7] = bad;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&lfull[u % kLook]);
            ++u;
            return true;
        };
        bool asked = false, ok = true;
        for (int n = 0, more = 1; more && ok && !s_abort; ++n) {
            ok = __all_sync(0xffffffffu, seg_ready(n));
            if (!ok) break;
            const Seg &sg = seg(n);
            const Tile ti = sg.t;
            const int b0 = sg.b0, b1 = sg.b1;
            more = sg.more;
            __syncwarp();
            if (lane == 0) seg_done(n);
            int parts = 0;
            for (int i = b0; i < b1 && ok; ++i) {
                const int blk = ti.block(i), p = blk * kCkKeys + lane * 16;
                int32_t pg = -1;
                int sl = -1;
                if (lane < kCkKeys / 16 && p < ti.hi && run_seen(a, ti, p)) {
                    const int en = a.c.page_of(p);
                    sl = p - en * a.c.page_size;
                    if (en < a.r.table_width) pg = a.r.table[(int64_t)ti.b * a.r.table_stride + en];
                }
                if (asked) ok = give();
                asked = true;
                page = pg;
                slot = sl;
                head = ti.h;
                e.left = ti.hi - blk * kCkKeys;
                e.blk = blk;
                e.seg = n;
                e.part = block_full(a, blk * kCkKeys, min(ti.minpos, ti.hi - 1), ti.maxpos) ? -1 : parts++;
            }
        }
        if (ok && asked) ok = give();
        e.part = -2;
        slot = -1;
        if (ok) give();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    if (s_abort && warp >= kCkMmaWarp && warp < kCkMmaWarp + 2 && lane == 0) {
        // a wait gave up: nothing may still write tensor memory when it is freed
        uint64_t *b = &sfull[warp - kCkMmaWarp];
        umma_commit(b);
        const long long t0 = clock64();
        while (clock64() - t0 < 10000000ll) {
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kCkMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename TA, int BITS, int D, int GS>
cudaError_t launch_chunk_t(const AttnArgs &a, cudaStream_t st) {
    using G = ChunkGeo<TA, BITS, D, GS>;
    auto kern = attn_chunk_kernel<TA, BITS, D, GS>;
    static bool configured[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = true;
    }
    const int grid = attn_num_sms();
    e = launch_pdl(kern, dim3((unsigned)grid), dim3(kCkThreads), G::SMEM, st, a);
    if (e != cudaSuccess) return e;
    return launch_attn_merge(std::is_same<TA, __half>::value, kCkRows, D, grid, kCkRows / 8, a, st);
}

template <typename TA>
cudaError_t launch_chunk_bits(int D, int bits, int gs, const AttnArgs &a, cudaStream_t st) {
#define LMOE_ATTN_CASE(B, DD, GG) \
    if (bits == B && D == DD && (B == 16 || gs == GG)) return launch_chunk_t<TA, B, DD, GG>(a, st);
    LMOE_ATTN_CASE(16, 64, 64)
    LMOE_ATTN_CASE(16, 128, 64)
    LMOE_ATTN_CASE(8, 64, 32)
    LMOE_ATTN_CASE(8, 64, 64)
    LMOE_ATTN_CASE(8, 128, 32)
    LMOE_ATTN_CASE(8, 128, 64)
    LMOE_ATTN_CASE(8, 128, 128)
    LMOE_ATTN_CASE(4, 64, 32)
    LMOE_ATTN_CASE(4, 64, 64)
    LMOE_ATTN_CASE(4, 128, 32)
    LMOE_ATTN_CASE(4, 128, 64)
    LMOE_ATTN_CASE(4, 128, 128)
#undef LMOE_ATTN_CASE
    return cudaErrorInvalidValue;
}

}  // namespace

size_t chunk_scratch_bytes(int D) {
    return (size_t)attn_num_sms() * (sizeof(MergeRec) + 2 * sizeof(float) * (size_t)kCkRows * (D + 2));
}

cudaError_t launch_attn_chunk(int act_f16, int head_dim, int bits, int group_size, const AttnArgs &a, cudaStream_t st) {
    return act_f16 ? launch_chunk_bits<__half>(head_dim, bits, group_size, a, st)
                   : launch_chunk_bits<__nv_bfloat16>(head_dim, bits, group_size, a, st);
}

}  // namespace lmoe
