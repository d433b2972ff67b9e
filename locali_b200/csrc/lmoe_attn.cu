// Attention of new token rows over the paged key/value cache.
//
// out = sum_j softmax_j(scale q . k_j) v_j over the positions a row sees, in
// one pass over the keys with the running maximum and sum of the softmax.
// One warp per (row, query head); lane l holds elements l, l + 32, ... of the
// head.
#include "lmoe_kernels.cuh"
#include "lmoe_kv.cuh"

namespace lmoe {

namespace {

template <typename TA, int BITS>
__device__ __forceinline__ float cached_value(const KvView &c, int which, int64_t row, int e) {
    if constexpr (BITS == 16) {
        return Act<TA>::to_f(reinterpret_cast<const uint16_t *>(c.kv[which])[row * (c.row_bytes / 2) + e]);
    } else {
        const uint8_t by = c.kv[which][row * c.row_bytes + e * BITS / 8];
        const uint32_t q = BITS == 8 ? by : (by >> (4 * (e & 1)) & 15u);
        const int64_t gi = row * c.groups + e / c.group_size;
        return fmaf(Act<TA>::to_f(c.scale[which][gi]), (float)q, Act<TA>::to_f(c.bias[which][gi]));
    }
}

template <typename TA, int BITS, int D>
__global__ void __launch_bounds__(256) attn_rows_kernel(const AttnArgs a) {
    constexpr int E = D / 32;
    pdl_wait();
    pdl_trigger();
    const int64_t wid = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (blockIdx.x == 0) a.r.validate(threadIdx.x, 256);
    if (wid >= (int64_t)a.r.n_rows * a.q_heads) return;
    const int r = (int)(wid / a.q_heads), h = (int)(wid % a.q_heads);
    int pos = 0;
    const int b = a.r.find(r, &pos);
    if (b < 0 && pos >= 0) return;  // no sequence's row
    const int hk = h / a.group;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = Act<TA>::to_f(a.q[r * a.q_tok_stride + h * a.q_head_stride + lane + 32 * i]) * a.scale_log2;
        o[i] = 0.0f;
    }
    bool any = false;
    if (b >= 0) {
        const int low = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        int j = a.sinks > 0 ? 0 : low;
        int cur = -1;
        int32_t page = -1;
        for (; j <= pos; ++j) {
            if (j < low && j >= a.sinks) j = low;
            if (j / a.c.page_size != cur) {
                cur = j / a.c.page_size;
                page = a.r.page(a.c, b, j);
            }
            if (page < 0) continue;
            any = true;
            const int64_t row = a.c.row(page, hk, j % a.c.page_size);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < E; ++i) s = fmaf(q[i], cached_value<TA, BITS>(a.c, 0, row, lane + 32 * i), s);
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            const float mn = fmaxf(m, s);
            const float f = mn == -INFINITY ? 1.0f : exp2f(m - mn), p = s == -INFINITY ? 0.0f : exp2f(s - mn);
            m = mn;
            l = l * f + p;
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = o[i] * f + p * cached_value<TA, BITS>(a.c, 1, row, lane + 32 * i);
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
        a.out[((int64_t)r * a.q_heads + h) * D + lane + 32 * i] = any ? Act<TA>::from_f(o[i] / l) : (uint16_t)0;
}

template <typename TA, int BITS, int D>
cudaError_t launch_rows(const AttnArgs &a, cudaStream_t st) {
    const int64_t warps = (int64_t)a.r.n_rows * a.q_heads;
    return launch_pdl(attn_rows_kernel<TA, BITS, D>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, st, a);
}

template <typename TA>
cudaError_t launch_bits(int D, int bits, const AttnArgs &a, cudaStream_t st) {
    if (D == 64) {
        if (bits == 16) return launch_rows<TA, 16, 64>(a, st);
        if (bits == 8) return launch_rows<TA, 8, 64>(a, st);
        return launch_rows<TA, 4, 64>(a, st);
    }
    if (bits == 16) return launch_rows<TA, 16, 128>(a, st);
    if (bits == 8) return launch_rows<TA, 8, 128>(a, st);
    return launch_rows<TA, 4, 128>(a, st);
}

}  // namespace

size_t attention_scratch_bytes(const KvRows &, int, int, int) { return 0; }

cudaError_t launch_attention(int act_f16, int head_dim, int bits, int, const AttnArgs &a, cudaStream_t st) {
    return act_f16 ? launch_bits<__half>(head_dim, bits, a, st) : launch_bits<__nv_bfloat16>(head_dim, bits, a, st);
}

}  // namespace lmoe
