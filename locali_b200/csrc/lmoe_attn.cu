// Attention of few rows (single tokens, a few drafted tokens) over the paged
// key/value cache, and the join of tiles cut over several blocks.
//
// out = sum_j softmax_j(scale q . k_j) v_j in one pass over the keys with the
// running reference (the maximum, shifted: Term in lmoe_attn.cuh) and sum of
// the softmax.  A tile's keys and values are read once.  On a B200 a 16-bit
// cache is bound by HBM (128 windowed sequences, 272 MB: 54 us, 5.0 of 6.5
// TB/s); codes by the instructions that make numbers of them (64 sequences of
// 4500 on average, 8 bits, 626 MB: 134 us, 4.7 TB/s, 64 % of the issue slots
// busy; 4 bits, 482 MB: 150 us, 3.2 TB/s).  Those are single launches; whole
// calls back to back, the join among them, take 68, 156 and 143 us.
//
// Work.  Tiles are 8 or 16 rows (tokens x query heads of one key/value head);
// the stream of their key blocks is cut evenly over the launch (Share in
// lmoe_attn.cuh).  Inside a launch block every warp takes key blocks of its
// own (KS positions, 4 KB of codes) and streams them through a private ring of
// shared-memory units with 16-byte cp.async, so warps never wait for one
// another inside a tile; their results meet once per tile.  Four launch blocks
// an SM keep 16 warps with two units each in flight (128 KB; three blocks where
// a tile has 16 rows), and one block's hand-over from tile to tile overlaps the
// others' streams.
//
// Registers are short: at heads of 128 the quantised instances spill, up to 114
// bytes of stores with tiles of 8 rows and 436 with 16 (-Xptxas -v), of which
// 0.1 % of the executed instructions are left (64 sequences, 8 bits).
//
// Arithmetic.  Both products are computed transposed, with the keys (values)
// as the 16-row operand of mma.m16n8k16 and the tile's 8 rows as its 8
// columns: S^T = K Q^T and O^T = V^T P^T.  With a handful of query heads per
// key/value head that halves the MMAs of the usual orientation, and the
// operands that come from memory can be assembled in registers straight from
// codes: the contraction order of K (the head dimension) and the row order of
// V^T are free, so a lane takes whole words of codes where they lie.
//
// Quantised keys are contracted as codes, one group of the head dimension
// after the other; scale and bias meet the group's fp32 sum, s (q . c) + b
// sum(q), so a key is never rounded (rounded to bf16 first, the keys were the
// largest part of a result's error, 2.9e-3 of 3.9e-3) and a code costs two
// instructions instead of four.  A constant added to the codes by the cheapest
// way to make them numbers (128 or 1024) is taken off with the bias (RawCode
// in lmoe_attn.cuh).  Values are dequantised to the 16-bit type: there a scale
// belongs to a position of the contraction.
#include "lmoe_attn.cuh"

namespace lmoe {

namespace {

constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kRowBlocksPerSm = 4;  // at most
constexpr int kRowTile = 2;         // what a tile costs besides its key blocks, in key blocks

template <int BITS, int D, int GS, int NT>
struct RowsGeo {
    static constexpr int R = 8 * NT;                               // rows of a tile
    static constexpr int RB = D * BITS / 8;                        // bytes of a head row
    static constexpr int KS = 4096 / RB < 64 ? 4096 / RB : 64;     // positions of a block
    static constexpr int NG = BITS == 16 ? 0 : D / GS;             // groups of a head row
    static constexpr int CB = KS * RB, SB = KS * NG * 2;           // code and scale bytes of a unit
    static constexpr int UB = CB + 2 * SB;                         // a unit: codes, scales, biases
    static constexpr int NU = 3;                                   // units of a warp's ring
    static constexpr int KT = KS / 16, MT = D / 16, QS = D / 16;   // 16-key steps, V^T row tiles, K steps
    static constexpr int MERGE = kRowWarps * R * (D + 4) * 4;      // per-warp results of a tile
    static constexpr int RING = kRowWarps * NU * UB;
    static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + kRowWarps * R * 8;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <int N>  // 1, 2 or 4 words
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[N]) {
    if constexpr (N == 1) {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a) : "memory");
    } else if constexpr (N == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a) : "memory");
    } else {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(a)
                     : "memory");
    }
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts_u16(uint32_t a, uint16_t v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
}

// Byte offset in a unit's codes of byte `o` of position `row`.  16-byte chunks
// are XOR-swizzled inside 128-byte lines so that a warp's reads fall in
// distinct banks: 16-bit rows by the row (ldmatrix of 8 rows); K codes, of
// which lane t of rows g = 0..7 reads the t-th quarter of a group (SEG bytes),
// so that the segments of as many rows as are read at once lie apart; V codes
// by the row pair (lane t reads rows 2t and 2t + 1).
template <int BITS, int D, int GS, int WHICH>
__host__ __device__ constexpr int unit_swizzle(int row) {
    constexpr int RB = D * BITS / 8, SEG = GS * BITS / 8;
    if (BITS == 16) return (row & 7) << 4;
    if (WHICH == 1) return RB == 32 ? (row & 4) << 3 : (row & 6) << 4;
    if (RB == 128) return SEG == 128 ? (row & 1) << 4 : SEG == 64 ? (row & 1) << 6 : (row & 3) << 5;
    if (RB == 64) return SEG == 64 ? 0 : SEG == 32 ? (row & 2) << 4 : (row & 6) << 3;
    return SEG == 32 ? 0 : (row & 4) << 2;
}
template <int BITS, int D, int GS, int WHICH>
__device__ __forceinline__ int unit_off(int row, int o) {
    return (row * (D * BITS / 8) + o) ^ unit_swizzle<BITS, D, GS, WHICH>(row);
}
// The same for row base + r, where `base` is known at compile time and has no
// bit of r, and base rows are whole 128-byte lines: `part` is unit_off(r, o).
template <int BITS, int D, int GS, int WHICH>
__device__ __forceinline__ uint32_t unit_at(int base, uint32_t part) {
    return base * (D * BITS / 8) + (part ^ unit_swizzle<BITS, D, GS, WHICH>(base));
}

template <typename TA, int BITS, int D, int GS, int NT>
__global__ void __launch_bounds__(kRowThreads, NT == 1 ? 4 : 3) attn_rows_kernel(const AttnArgs a) {
    using G = RowsGeo<BITS, D, GS, NT>;
    constexpr int R = G::R, KS = G::KS, KT = G::KT, MT = G::MT, QS = G::QS, NG = G::NG, RB = G::RB;
    constexpr bool Q = BITS != 16;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long s_plan[kRowWarps + 4];
    __shared__ float s_qs[kRowWarps][NG ? NG : 1][R];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = smem_u32(sm) + warp * (G::NU * G::UB);
    float *s_o = reinterpret_cast<float *>(sm);
    float *s_ml = reinterpret_cast<float *>(sm + (G::SMEM - kRowWarps * R * 8));
    MergeRec *rec = reinterpret_cast<MergeRec *>(a.scratch) + blockIdx.x;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0) a.r.validate(tid, kRowThreads);
    Share sh;
    Cursor<R, KS, kRowTile> cur;
    // a run of at least one key block for each warp
    const bool work = find_share<R, KS, kRowTile, kRowThreads, false>(a, kRowTile + kRowWarps, s_plan, sh, cur);
    if (tid == 0) rec->parts = 0;
    if (!work) return;
    const float sc = a.scale_log2 / RawCode<TA, BITS>::kDown;

    for (;;) {
        const Tile &t = cur.t;
        const int b0 = cur.b0, b1 = cur.b1;

        // ---- the tile's rows as the column operand of S^T, in the order of K's words
        uint32_t qf[NT][QS][2];
        int pos[NT][2];  // positions of this lane's two columns' rows; -1: no row
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = t.rt * R + n * 8 + g;  // in the sequence's rows
            const bool in = row < t.n * a.group;
            const int tok = a.per_group(row);
            const uint16_t *q = a.q + (int64_t)(t.row0 + tok) * a.q_tok_stride +
                                (int64_t)(t.h * a.group + row - tok * a.group) * a.q_head_stride;
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                uint32_t x0 = 0, x1 = 0;
                if constexpr (BITS == 16) {
                    if (in) {
                        x0 = *reinterpret_cast<const uint32_t *>(q + 16 * s + 2 * t4);
                        x1 = *reinterpret_cast<const uint32_t *>(q + 16 * s + 8 + 2 * t4);
                    }
                } else {
                    // step s: word (or half of a word's code pairs) s % SPG of
                    // the lane's quarter of group s / SPG
                    constexpr int SPG = GS / 16;
                    const int d0 = (s / SPG) * GS + t4 * (GS / 4) + (BITS == 8 ? 4 * (s % SPG) : 8 * (s % SPG >> 1) + 2 * (s & 1));
                    uint2 v = make_uint2(0u, 0u);
                    if (in) {
                        v.x = *reinterpret_cast<const uint32_t *>(q + d0);
                        v.y = *reinterpret_cast<const uint32_t *>(q + d0 + (BITS == 8 ? 2 : 4));
                    }
                    // 8 bits: codes (c0, c2), (c1, c3); 4 bits: (c0, c4), (c1, c5), then (c2, c6), (c3, c7)
                    x0 = __byte_perm(v.x, v.y, 0x5410);
                    x1 = __byte_perm(v.x, v.y, 0x7632);
                }
                qf[n][s][0] = x0;
                qf[n][s][1] = x1;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int rc = t.rt * R + n * 8 + 2 * t4 + c;
                pos[n][c] = rc < t.n * a.group ? t.first + a.per_group(rc) : -1;
            }
        }
        // sums of the tile's rows over the groups, in shared memory: registers are short
        if constexpr (Q) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) {
                    float x = 0.0f;
#pragma unroll
                    for (int s = gi * (GS / 16); s < (gi + 1) * (GS / 16); ++s)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            x += Act<TA>::to_f((uint16_t)(qf[n][s][h] & 0xFFFFu)) + Act<TA>::to_f((uint16_t)(qf[n][s][h] >> 16));
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    __syncwarp();
                    if (t4 == 0) s_qs[warp][gi][n * 8 + g] = x;
                }
            __syncwarp();
        }
        float o[NT][MT][4], m[NT][2], l[NT][2];
        bool seen[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[n][c] = -INFINITY;
                l[n][c] = 0.0f;
                seen[n][c] = false;
            }
        }

        // ---- this warp's blocks of [b0, b1), as units K, V, K, V, ...
        const int nb = b0 + warp < b1 ? (b1 - b0 - warp + kRowWarps - 1) / kRowWarps : 0;
        // Head row (of all pages') where 16-position run `lane` of block i of
        // the warp's begins; -2: no such positions, or none
        // that a row sees; -1: no page.
        auto runs_of = [&](int i) -> long long {
            long long r = lane < KT ? -2 : 0;
            if (lane < KT && i < nb) {
                const int p = t.block(b0 + warp + i * kRowWarps) * KS + lane * 16;
                if (p < t.hi && run_seen(a, t, p)) {
                    const int32_t pg = a.r.page(a.c, t.b, p);
                    r = pg < 0 ? -1 : a.c.row(pg, t.h, a.c.slot_of(p));
                }
            }
            return r;
        };
        auto issue = [&](auto which, int i, long long runs, int slot) {
            constexpr int W = decltype(which)::value;
            constexpr int RPI = 512 / RB;  // rows of one copy instruction of the warp
            if (i < nb) {
                const int k0 = t.block(b0 + warp + i * kRowWarps) * KS;
                const uint32_t u = ring + slot * G::UB;
                const int r0 = lane / (RB / 16), c0 = lane % (RB / 16);
                const uint32_t part = unit_off<BITS, D, GS, W>(r0, c0 * 16);
                const bool all = k0 + KS <= t.hi && !__any_sync(0xffffffffu, runs < 0);
                const uint8_t *const kv = a.c.kv[W] + lane * 16;
                if (all) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        const uint8_t *src = kv + __shfl_sync(0xffffffffu, runs, kt) * RB;
#pragma unroll
                        for (int it = 0; it < 16 / RPI; ++it)
                            cp16(u + unit_at<BITS, D, GS, W>(kt * 16 + it * RPI, part), src + it * 512);
                    }
                } else {
#pragma unroll 1
                    for (int kt = 0; kt < KT; ++kt) {
                        const long long run = __shfl_sync(0xffffffffu, runs, kt);
#pragma unroll 1
                        for (int it = 0; it < 16 / RPI; ++it) {
                            const int row = kt * 16 + it * RPI + r0;
                            const bool in = run >= 0 && k0 + row < t.hi;
                            cp16z(u + unit_off<BITS, D, GS, W>(row, c0 * 16), in ? kv + run * RB + it * 512 : a.c.kv[W],
                                  in ? 16 : 0);
                        }
                    }
                }
                if constexpr (Q) {
                    constexpr int CPR = 2 * NG;  // 16-byte chunks of a run's scales
                    static_assert(CPR * KT <= 32, "one chunk a lane");
                    const int run = min(lane / CPR, KT - 1), c = lane % CPR;
                    const long long r = __shfl_sync(0xffffffffu, runs, run);
                    if (lane < CPR * KT) {
                        int bytes = min(16, max(0, (t.hi - k0 - run * 16) * NG * 2 - c * 16));
                        if (r < 0) bytes = 0;
                        const long long off = bytes ? r * NG + c * 8 : 0;
                        cp16z(u + G::CB + lane * 16, a.c.scale[W] + off, bytes);
                        cp16z(u + G::CB + G::SB + lane * 16, a.c.bias[W] + off, bytes);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        using K0 = std::integral_constant<int, 0>;
        using V1 = std::integral_constant<int, 1>;
        long long pg_cur = runs_of(0), pg_next = runs_of(1), pg_far = runs_of(2);
        issue(K0{}, 0, pg_cur, 0);
        issue(V1{}, 0, pg_cur, 1);
        issue(K0{}, 1, pg_next, 2);
        int ks = 0;  // ring slot of the block's keys; its values follow
        for (int i = 0; i < nb; ++i) {
            const int vs = ks + 1 >= G::NU ? ks + 1 - G::NU : ks + 1;
            const int k0 = t.block(b0 + warp + i * kRowWarps) * KS;
            const uint32_t bad = __ballot_sync(0xffffffffu, pg_cur == -1);  // runs without a page
            // every row of the tile sees every position of the block
            const bool full = !bad && k0 + KS - 1 <= t.minpos && k0 + KS <= t.hi &&
                              (a.window == 0 || k0 > (long long)t.maxpos - a.window || k0 + KS <= a.sinks);

            // ---- S^T = K Q^T
            cp_wait<G::NU - 1>();
            __syncwarp();
            float s[KT][NT][4];
            const uint32_t ku = ring + ks * G::UB;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kt][n][e] = 0.0f;
            if constexpr (BITS == 16) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const uint32_t part = unit_off<16, D, GS, 0>(lane & 15, (lane >> 4) * 16);
#pragma unroll
                    for (int x = 0; x < QS; ++x) {
                        uint32_t f[4];
                        ldsm4(ku + kt * 16 * RB + (part ^ (x * 32)), f);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            Act<TA>::mma(s[kt][n], f[0], f[1], f[2], f[3], qf[n][x][0], qf[n][x][1]);
                    }
                }
            } else {
                constexpr int SEG = GS * BITS / 8, WPG = SEG / 16;  // bytes of a group, words of a lane's quarter
                constexpr int WV = WPG < 4 ? WPG : 4;               // read at once
                using RC = RawCode<TA, BITS>;
                const uint32_t part = unit_off<BITS, D, GS, 0>(g, t4 * (SEG / 4));
                const uint32_t spart = ku + G::CB + g * NG * 2;
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) {
                    float2 qs[NT];  // of the lane's two columns
#pragma unroll
                    for (int n = 0; n < NT; ++n) qs[n] = *reinterpret_cast<const float2 *>(&s_qs[warp][gi][n * 8 + 2 * t4]);
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        float sf[2], bf[2], acc[NT][4];
                        uint32_t w[2][WPG];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int x = 0; x < WPG; x += WV) {
                                uint32_t y[WV];
                                lds_words<WV>(ku + (kt * 16 + 8 * h) * RB + (part ^ (gi * SEG + x * 4)), y);
#pragma unroll
                                for (int e = 0; e < WV; ++e) w[h][x + e] = y[e];
                            }
                            const uint32_t so = spart + (kt * 16 + 8 * h) * NG * 2 + gi * 2;
                            const float sv = Act<TA>::to_f((uint16_t)lds_u16(so)), bv = Act<TA>::to_f((uint16_t)lds_u16(so + G::SB));
                            // a scale or bias that is no number makes the key's score none: 0 times it is none either
                            bf[h] = fmaf(bv, RC::kDown, fmaf(bv, 0.0f, sv * 0.0f));
                            if constexpr (RC::kOffset != 0.0f) bf[h] = fmaf(-RC::kOffset * RC::kDown, sv, bf[h]);
                            sf[h] = sv * (RC::kDown / RC::kUnit);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
#pragma unroll
                        for (int x = 0; x < WPG; ++x)
#pragma unroll
                            for (int hf = 0; hf < (BITS == 4 ? 2 : 1); ++hf) {
                                const int st = gi * (GS / 16) + (BITS == 4 ? 2 * x + hf : x);
                                const uint32_t a0 = RC::pair(w[0][x], 2 * hf), a1 = RC::pair(w[1][x], 2 * hf);
                                const uint32_t a2 = RC::pair(w[0][x], 2 * hf + 1), a3 = RC::pair(w[1][x], 2 * hf + 1);
#pragma unroll
                                for (int n = 0; n < NT; ++n)
                                    Act<TA>::mma(acc[n], a0, a1, a2, a3, qf[n][st][0], qf[n][st][1]);
                            }
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s[kt][n][e] = fmaf(sf[e >> 1], acc[n][e], fmaf(bf[e >> 1], e & 1 ? qs[n].y : qs[n].x, s[kt][n][e]));
                    }
                }
            }
            __syncwarp();
            issue(V1{}, i + 1, pg_next, ks);  // the keys' slot is free

            // ---- softmax over the block: mask, maximum, terms
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kt][n][e] *= sc;
            if (!full) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = k0 + kt * 16 + g + 8 * (e >> 1), p = pos[n][e & 1];
                            const bool see = j <= p && j < t.hi && !(bad >> kt & 1u) &&
                                             (a.window == 0 || p - j < a.window || j < a.sinks);
                            seen[n][e & 1] |= see;
                            if (!see) s[kt][n][e] = -INFINITY;
                        }
            }
            bool moved = false;
            float mu[NT][2], f[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = max_nan(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
                    for (int kt = 1; kt < KT; ++kt) x = max_nan(x, max_nan(s[kt][n][c], s[kt][n][c + 2]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, d));
                    x = max_nan(m[n][c], x - Term<TA, false>::kSet);
                    if (full) seen[n][c] = true;
                    mu[n][c] = x == -INFINITY ? 0.0f : x;
                    f[n][c] = ex2(m[n][c] - mu[n][c]);
                    moved |= !(x == m[n][c]);
                    m[n][c] = x;
                }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    l[n][0] *= f[n][0];
                    l[n][1] *= f[n][1];
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        o[n][x][0] *= f[n][0];
                        o[n][x][1] *= f[n][1];
                        o[n][x][2] *= f[n][0];
                        o[n][x][3] *= f[n][1];
                    }
                }
            }
            uint32_t pf[KT][NT][2];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = ex2(s[kt][n][e] - mu[n][e & 1]);
                    l[n][0] += p[0] + p[2];
                    l[n][1] += p[1] + p[3];
                    pf[kt][n][0] = movm(Act<TA>::pack2(p[0], p[1]));
                    pf[kt][n][1] = movm(Act<TA>::pack2(p[2], p[3]));
                }

            // ---- O^T += V^T P^T
            cp_wait<G::NU - 1>();
            __syncwarp();
            const uint32_t vu = ring + vs * G::UB;
            if (!full) {
                // A value that is no number must not reach the rows that do
                // not see its position (0 times it is no number either): it
                // is added here to those that do and taken out of the unit.
                constexpr int W4 = RB / 4, SW = NG;
                bool odd = false;
                if constexpr (Q) {
                    for (int i2 = lane; i2 < KS * SW; i2 += 32) {
                        const uint32_t x = lds_u16(vu + G::CB + i2 * 2), y = lds_u16(vu + G::CB + G::SB + i2 * 2);
                        odd |= group_past_type<TA, BITS>(x, y);
                    }
                } else {
                    for (int i2 = lane; i2 < KS * W4; i2 += 32) {
                        uint32_t x[1];
                        lds_words<1>(vu + i2 * 4, x);
                        odd |= nonfinite16<TA>(x[0]) || nonfinite16<TA>(x[0] >> 16);
                    }
                }
                if (__any_sync(0xffffffffu, odd)) {
                    for (int k = 0; k < KS; ++k) {
                        const int j = k0 + k;
#pragma unroll
                        for (int x = 0; x < MT; ++x)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                // the lane's row of V^T (see the products below)
                                const int dim = Q ? (D / 8) * g + h * (D / 16) + x : 16 * x + 8 * h + g;
                                float v;
                                if constexpr (Q) {
                                    const int byte = dim * BITS / 8;
                                    uint32_t w[1];
                                    lds_words<1>(vu + unit_off<BITS, D, GS, 1>(k, byte & ~3), w);
                                    const uint32_t code = w[0] >> (dim * BITS % 32) & ((1u << BITS) - 1u);
                                    const uint32_t so = vu + G::CB + (k * SW + dim / GS) * 2;
                                    v = code_value<TA, BITS>(code, lds_u16(so), lds_u16(so + G::SB));
                                } else {
                                    v = Act<TA>::to_f((uint16_t)lds_u16(vu + unit_off<16, D, GS, 1>(k, dim * 2)));
                                }
                                if (past_type<TA>(v)) {
                                    v *= INFINITY;
#pragma unroll
                                    for (int n = 0; n < NT; ++n)
#pragma unroll
                                        for (int c = 0; c < 2; ++c) {
                                            const int p = pos[n][c];
                                            if (j <= p && (a.window == 0 || p - j < a.window || j < a.sinks))
                                                o[n][x][2 * h + c] += v;
                                        }
                                }
                            }
                    }
                    __syncwarp();
                    if constexpr (Q) {
                        // single codes become code 0, groups of which that is no number either become zero
#pragma unroll 1
                        for (int i2 = lane; i2 < KS * W4; i2 += 32) {
                            const int k = i2 / W4, byte = i2 % W4 * 4;
                            const uint32_t wa = vu + unit_off<BITS, D, GS, 1>(k, byte);
                            const uint32_t so = vu + G::CB + (k * SW + byte * 8 / BITS / GS) * 2;
                            const uint32_t x = lds_u16(so), y = lds_u16(so + G::SB);
                            if (!group_past_type<TA, BITS>(x, y)) continue;
                            uint32_t w[1];
                            lds_words<1>(wa, w);
#pragma unroll 1
                            for (int sh = 0; sh < 32; sh += BITS)
                                if (past_type<TA>(code_value<TA, BITS>(w[0] >> sh & ((1u << BITS) - 1u), x, y)))
                                    w[0] &= ~(((1u << BITS) - 1u) << sh);
                            sts_u16(wa, (uint16_t)w[0]);
                            sts_u16(wa + 2, (uint16_t)(w[0] >> 16));
                        }
                        __syncwarp();
                        for (int i2 = lane; i2 < KS * SW; i2 += 32) {
                            const uint32_t sa = vu + G::CB + i2 * 2;
                            if (past_type<TA>(code_value<TA, BITS>(0u, lds_u16(sa), lds_u16(sa + G::SB)))) {
                                sts_u16(sa, 0);
                                sts_u16(sa + G::SB, 0);
                            }
                        }
                    } else {
                        for (int i2 = lane; i2 < KS * W4 * 2; i2 += 32)
                            if (nonfinite16<TA>(lds_u16(vu + i2 * 2))) sts_u16(vu + i2 * 2, 0);
                    }
                    __syncwarp();
                }
            }
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                if constexpr (BITS == 16) {
                    const uint32_t part = unit_off<16, D, GS, 1>((lane & 7) + (lane >> 4) * 8, (lane >> 3 & 1) * 16);
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        uint32_t f4[4];
                        ldsm4t(vu + kt * 16 * RB + (part ^ (x * 32)), f4);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            Act<TA>::mma(o[n][x], f4[0], f4[1], f4[2], f4[3], pf[kt][n][0], pf[kt][n][1]);
                    }
                } else {
                    // lane: dims (D / 8) g .. of positions 2 t4, 2 t4 + 1 (first
                    // half of the step) and 8 behind them; row g of row tile x
                    // is dim (D / 8) g + x, row g + 8 is D / 16 further
                    constexpr int WL = RB / 8 / 4;  // words of the lane's dims
                    uint32_t u[2][WL][2], s2[2], b2[2];
                    const uint32_t part0 = unit_off<BITS, D, GS, 1>(2 * t4, g * (RB / 8));
                    const uint32_t part1 = unit_off<BITS, D, GS, 1>(2 * t4 + 1, g * (RB / 8));
                    const uint32_t spart = vu + G::CB + (2 * t4 * NG + (D / 8) * g / GS) * 2;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w0[WL], w1[WL];
                        lds_words<WL>(vu + unit_at<BITS, D, GS, 1>(kt * 16 + 8 * h, part0), w0);
                        lds_words<WL>(vu + unit_at<BITS, D, GS, 1>(kt * 16 + 8 * h, part1), w1);
#pragma unroll
                        for (int x = 0; x < WL; ++x) {
                            u[h][x][0] = __byte_perm(w0[x], w1[x], 0x5410);
                            u[h][x][1] = __byte_perm(w0[x], w1[x], 0x7632);
                        }
                        const uint32_t so = spart + (kt * 16 + 8 * h) * NG * 2;
                        s2[h] = Pair<TA>::template scale<BITS>(lds_u16(so) | lds_u16(so + NG * 2) << 16);
                        b2[h] = lds_u16(so + G::SB) | lds_u16(so + G::SB + NG * 2) << 16;
                    }
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        // dims x and MT + x of the lane's: half-word and code in it
                        constexpr int CH = 16 / BITS;  // codes of a half-word
                        const int i0 = x / CH, i1 = (MT + x) / CH, j = x % CH;
                        const uint32_t a0 = code_pair<TA, BITS>(u[0][i0 >> 1][i0 & 1], j, s2[0], b2[0]);
                        const uint32_t a1 = code_pair<TA, BITS>(u[0][i1 >> 1][i1 & 1], j, s2[0], b2[0]);
                        const uint32_t a2 = code_pair<TA, BITS>(u[1][i0 >> 1][i0 & 1], j, s2[1], b2[1]);
                        const uint32_t a3 = code_pair<TA, BITS>(u[1][i1 >> 1][i1 & 1], j, s2[1], b2[1]);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            Act<TA>::mma(o[n][x], a0, a1, a2, a3, pf[kt][n][0], pf[kt][n][1]);
                    }
                }
            }
            __syncwarp();
            pg_cur = pg_next;
            pg_next = pg_far;
            issue(K0{}, i + 2, pg_next, vs);  // the values' slot is free
            pg_far = runs_of(i + 3);
            ks = ks == 0 ? 2 : ks - 1;  // two units on, of three
        }
        cp_wait<0>();
        __syncthreads();  // every warp's ring is free: the results of the warps meet there

        // ---- join the warps
        const bool whole = b0 == 0 && b1 == t.nblk;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[n][c];
                uint32_t sn = seen[n][c];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    x += __shfl_xor_sync(0xffffffffu, x, d);
                    sn |= __shfl_xor_sync(0xffffffffu, sn, d);
                }
                // only scores of -inf: the softmax is no number, unless other
                // parts of the tile's keys hold larger ones
                if (sn && m[n][c] == -INFINITY) x = __uint_as_float(0x7FC00000u);
                if (g == 0) {
                    s_ml[(warp * R + n * 8 + 2 * t4 + c) * 2] = m[n][c];
                    s_ml[(warp * R + n * 8 + 2 * t4 + c) * 2 + 1] = x;
                }
#pragma unroll
                for (int x2 = 0; x2 < MT; ++x2)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int dim = Q ? (D / 8) * g + h * (D / 16) + x2 : 16 * x2 + 8 * h + g;
                        s_o[(warp * R + n * 8 + 2 * t4 + c) * (D + 4) + dim] = o[n][x2][2 * h + c];
                    }
            }
        __syncthreads();
        float *part = part_ptr(a, gridDim.x, part_floats<R, D>(), blockIdx.x, b0 == 0 ? 1 : 0);
        for (int i = tid; i < R * (D / 4); i += kRowThreads) {
            const int row = i / (D / 4), d = (i % (D / 4)) * 4;
            float mm = -INFINITY, ll = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) mm = max_nan(mm, s_ml[(w * R + row) * 2]);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                const float mw = s_ml[(w * R + row) * 2];
                if (mw == -INFINITY && mm != -INFINITY) continue;
                const float x = mw == -INFINITY ? 1.0f : ex2(mw - mm);
                const float4 v = *reinterpret_cast<const float4 *>(s_o + (w * R + row) * (D + 4) + d);
                ll += x * s_ml[(w * R + row) * 2 + 1];
                acc.x += x * v.x;
                acc.y += x * v.y;
                acc.z += x * v.z;
                acc.w += x * v.w;
            }
            if (!whole) {
                *reinterpret_cast<float4 *>(part + row * D + d) = acc;
                if (d == 0) {
                    part[R * D + row * 2] = mm;
                    part[R * D + row * 2 + 1] = ll;
                }
            } else if (row < t.rows) {
                const int rr = t.rt * R + row, tok = a.per_group(rr);
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                uint2 v;
                v.x = Act<TA>::pack2(acc.x * inv, acc.y * inv);
                v.y = Act<TA>::pack2(acc.z * inv, acc.w * inv);
                *reinterpret_cast<uint2 *>(a.out + ((int64_t)(t.row0 + tok) * a.q_heads + t.h * a.group + rr -
                                                    tok * a.group) * D + d) = v;
            }
        }
        const int shared = cur.shared(sh, blockIdx.x);
        if (tid == 0 && shared) {
            rec->out0 = t.row0;
            rec->row = t.rt * R;
            rec->rows_h = t.rows | t.h << 16;
            rec->parts = shared;
        }
        __syncthreads();
        if (!cur.next(a)) break;
    }
}

// Joins the parts of the tiles that were cut: block (c, y) the tile that goes
// on behind launch block c's run; row by row (rows split over y), a warp's
// lanes the head dimension, the block's warps every 8th part.
template <typename TA, int R, int D>
__global__ void __launch_bounds__(256) attn_merge_kernel(const AttnArgs a, int grid) {
    constexpr int V = D / 32;  // elements of a lane
    __shared__ float s_m[8], s_l[8], s_o[8][D];
    pdl_wait();
    pdl_trigger();
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const MergeRec rec = reinterpret_cast<const MergeRec *>(a.scratch)[c];
    if (rec.parts < 2) return;
    const int rows = rec.rows_h & 0xFFFF, h = rec.rows_h >> 16;
    const float *first = part_ptr(a, grid, part_floats<R, D>(), c, 1);
    const size_t pf = part_floats<R, D>();
    auto part = [&](int i) { return i == 0 ? first : first + (size_t)(2 * i - 1) * pf; };
    const bool wide = rec.parts > 8;  // many parts: all warps on one row; few: a row each
    for (int row = blockIdx.y * (wide ? 1 : 8) + (wide ? 0 : warp); row < rows; row += gridDim.y * (wide ? 1 : 8)) {
        float mm = -INFINITY, ll = 0.0f, acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        const int i0 = wide ? warp : 0, step = wide ? 8 : 1;
        for (int i = i0 + lane * step; i < rec.parts; i += 32 * step) mm = max_nan(mm, part(i)[R * D + row * 2]);
#pragma unroll
        for (int d = 16; d; d >>= 1) mm = max_nan(mm, __shfl_xor_sync(0xffffffffu, mm, d));
#pragma unroll 4
        for (int i = i0; i < rec.parts; i += step) {
            const float *p = part(i);
            const float mi = p[R * D + row * 2], li = p[R * D + row * 2 + 1];
            float x[V];
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = p[row * D + v * 32 + lane];
            if (mi == -INFINITY && mm != -INFINITY) continue;
            const float w = mi == -INFINITY ? 1.0f : ex2(mi - mm);
            ll += w * li;
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] += w * x[v];
        }
        if (wide) {
            if (lane == 0) {
                s_m[warp] = mm;
                s_l[warp] = ll;
            }
#pragma unroll
            for (int v = 0; v < V; ++v) s_o[warp][v * 32 + lane] = acc[v];
            __syncthreads();
            if (warp == 0) {
                mm = -INFINITY;
                ll = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) mm = max_nan(mm, s_m[w]);
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] = 0.0f;
                for (int w = 0; w < 8; ++w) {
                    if (s_m[w] == -INFINITY && mm != -INFINITY) continue;
                    const float x = s_m[w] == -INFINITY ? 1.0f : ex2(s_m[w] - mm);
                    ll += x * s_l[w];
#pragma unroll
                    for (int v = 0; v < V; ++v) acc[v] += x * s_o[w][v * 32 + lane];
                }
            }
            __syncthreads();
            if (warp != 0) continue;
        }
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        const int rr = rec.row + row, tok = a.per_group(rr);
        uint16_t *out = a.out + ((int64_t)(rec.out0 + tok) * a.q_heads + h * a.group + rr - tok * a.group) * D;
#pragma unroll
        for (int v = 0; v < V; ++v) out[v * 32 + lane] = Act<TA>::from_f(acc[v] * inv);
    }
}

template <typename TA, int BITS, int D, int GS, int NT>
cudaError_t launch_rows_t(const AttnArgs &a, cudaStream_t st) {
    using G = RowsGeo<BITS, D, GS, NT>;
    auto kern = attn_rows_kernel<TA, BITS, D, GS, NT>;
    // launch blocks that fit on an SM at once, by device; the whole launch is resident
    static int per_sm[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    int fit = dev < 64 ? per_sm[dev] : 0;
    if (fit == 0) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, kRowThreads, G::SMEM);
        if (e != cudaSuccess) return e;
        fit = min(max(fit, 1), kRowBlocksPerSm);
        if (dev < 64) per_sm[dev] = fit;
    }
    const int grid = attn_num_sms() * fit;
    e = launch_pdl(kern, dim3((unsigned)grid), dim3(kRowThreads), G::SMEM, st, a);
    if (e != cudaSuccess) return e;
    // few tiles, each cut into many parts: a merge block for each row
    const int y = (long long)a.r.n_seqs * a.c.kv_heads * 8 < grid ? G::R : 1;
    return launch_attn_merge(std::is_same<TA, __half>::value, G::R, D, grid, y, a, st);
}

template <typename TA, int BITS, int D, int GS>
cudaError_t launch_nt(int nt, const AttnArgs &a, cudaStream_t st) {
    return nt == 1 ? launch_rows_t<TA, BITS, D, GS, 1>(a, st) : launch_rows_t<TA, BITS, D, GS, 2>(a, st);
}

template <typename TA>
cudaError_t launch_rows(int D, int bits, int gs, int nt, const AttnArgs &a, cudaStream_t st) {
#define LMOE_ATTN_CASE(B, DD, GG) \
    if (bits == B && D == DD && (B == 16 || gs == GG)) return launch_nt<TA, B, DD, GG>(nt, a, st);
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

// tiles of 8 rows while the sequences have that many on average, else of 16
int rows_nt(const KvRows &r, int group) { return (long long)r.n_rows * group <= 8ll * r.n_seqs ? 1 : 2; }

// Chunks on average: the tcgen05 kernel's tiles of 256 rows.
bool use_chunk(const KvRows &r, int group) { return (long long)r.n_rows * group > 16ll * r.n_seqs; }

}  // namespace

int attn_num_sms() {
    static int sms[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (sms[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
        sms[dev] = n;
    }
    return sms[dev];
}

cudaError_t launch_attn_merge(int act_f16, int R, int D, int grid, int y, const AttnArgs &a, cudaStream_t st) {
    const dim3 g((unsigned)grid, (unsigned)y), b(256);
#define LMOE_MERGE_CASE(RR, DD)                                                                       \
    if (R == RR && D == DD)                                                                           \
        return act_f16 ? launch_pdl(attn_merge_kernel<__half, RR, DD>, g, b, 0, st, a, grid)          \
                       : launch_pdl(attn_merge_kernel<__nv_bfloat16, RR, DD>, g, b, 0, st, a, grid);
    LMOE_MERGE_CASE(8, 64)
    LMOE_MERGE_CASE(8, 128)
    LMOE_MERGE_CASE(16, 64)
    LMOE_MERGE_CASE(16, 128)
    LMOE_MERGE_CASE(256, 64)
    LMOE_MERGE_CASE(256, 128)
#undef LMOE_MERGE_CASE
    return cudaErrorInvalidValue;
}

size_t attention_scratch_bytes(const KvRows &r, int, int group, int D) {
    if (r.n_rows == 0 || r.n_seqs == 0) return 0;
    if (use_chunk(r, group)) return chunk_scratch_bytes(D);
    const int nt = rows_nt(r, group), grid = attn_num_sms() * kRowBlocksPerSm;
    return (size_t)grid * (sizeof(MergeRec) + 2 * sizeof(float) * (size_t)(8 * nt) * (D + 2));
}

cudaError_t launch_attention(int act_f16, int head_dim, int bits, int group_size, const AttnArgs &a, cudaStream_t st) {
    if (use_chunk(a.r, a.group)) return launch_attn_chunk(act_f16, head_dim, bits, group_size, a, st);
    const int nt = rows_nt(a.r, a.group);
    return act_f16 ? launch_rows<__half>(head_dim, bits, group_size, nt, a, st)
                   : launch_rows<__nv_bfloat16>(head_dim, bits, group_size, nt, a, st);
}

}  // namespace lmoe
