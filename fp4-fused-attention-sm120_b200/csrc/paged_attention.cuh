// paged_attention.cuh -- attention of one new token per sequence over the
// paged FP4 key / FP16 value cache (sm_100a).
//
//     z_j = scale * Qq . Kq_j,   o = sum_j exp(z_j) v_j / sum_j exp(z_j),
// j over the first seq_lens[b] tokens of sequence b, Qq the query quantised
// as the forward quantises it, Kq the cache's keys.  A sequence of length 0
// gives o = 0 and log-sum-exp +inf, as a row without visible keys does in the
// forward.
#pragma once

#include <cuda_fp16.h>
#include <cstdint>

#include "paged.cuh"

namespace fp4attn {

struct PagedArgs {
    const void* q;
    int64_t qb, qh;       // element strides of batch and head
    int batch, q_heads, group;
    CacheView c;
    TableView t;
    const int32_t* seq_lens;
    float scale_log2;     // softmax scale * log2(e)
    int ocp;
    void* out;            // [batch][q_heads][head_dim]
    float* lse;           // [batch][q_heads] or null
};

// One block per (query head, sequence): 128 keys a step, one per thread, the
// running maximum and sum in FP32, then one output column per thread.
template <typename InT, typename OutT, int D>
__global__ void __launch_bounds__(128) paged_attention_simple_kernel(const PagedArgs a)
{
    __shared__ float sq[D];
    __shared__ float sp[128];
    __shared__ int spage[128];
    __shared__ float red[8];
    const int hq = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, kvh = hq / a.group;
    int len = a.seq_lens[b];
    const int64_t most = static_cast<int64_t>(a.t.max_pages) * a.c.page_size;
    if (len < 0 || len > most) {
        if (tid == 0) record_index_error(kIndexLength, len);
        len = len < 0 ? 0 : static_cast<int>(most);
    }
    if (tid < D / 32) {
        const InT* q = static_cast<const InT*>(a.q) + b * a.qb + hq * a.qh + tid * 32;
        float v[32];
        for (int i = 0; i < 32; i++) v[i] = to_float(q[i]);
        uint4 packed;
        const uint32_t sb = encode32<InT>(v, a.ocp, packed);
        const float sc = scale_value(sb == 255u ? 254u : sb);
        const uint32_t w[4] = {packed.x, packed.y, packed.z, packed.w};
        for (int i = 0; i < 32; i++) sq[tid * 32 + i] = e2m1_value((w[i / 8] >> (4 * (i % 8))) & 15u) * sc;
    }
    __syncthreads();
    constexpr int C = (D + 127) / 128;
    float m = -INFINITY, l = 0.f, o[C] = {};
    for (int t0 = 0; t0 < len; t0 += 128) {
        const int pos = t0 + tid;
        float z = -INFINITY;
        int page = -1;
        if (pos < len) page = page_of(a.c, a.t, b, pos);
        if (page >= 0) {
            const int64_t row = static_cast<int64_t>(kvh) * a.c.page_size + (pos & (a.c.page_size - 1));
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.c.k_codes + page * a.c.k_codes_stride + row * (D / 2));
            const uint8_t* scales = a.c.k_scales + page * a.c.k_scales_stride + row * (D / 32);
            float s = 0.f;
            for (int blk = 0; blk < D / 32; blk++) {
                float p = 0.f;
                for (int w = 0; w < 4; w++) {
                    const uint32_t cw = codes[blk * 4 + w];
                    for (int j = 0; j < 8; j++) p = fmaf(e2m1_value((cw >> (4 * j)) & 15u), sq[blk * 32 + w * 8 + j], p);
                }
                s = fmaf(p, scale_value(scales[blk]), s);
            }
            z = s * a.scale_log2;
        }
        float mx = z;
        for (int i = 16; i; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, i));
        if (tid % 32 == 0) red[tid / 32] = mx;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = mn == -INFINITY ? 0.f : mn;
        const float p = exp2f(z - base), alpha = exp2f(m - base);
        sp[tid] = p;
        spage[tid] = page;
        float sum = p;
        for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
        if (tid % 32 == 0) red[4 + tid / 32] = sum;
        __syncthreads();
        l = l * alpha + (red[4] + red[5] + red[6] + red[7]);
        m = mn;
        for (int c = 0; c < C; c++) o[c] *= alpha;
        for (int j = 0; j < min(128, len - t0); j++) {
            if (spage[j] < 0) continue;
            const __half* v = reinterpret_cast<const __half*>(reinterpret_cast<const uint8_t*>(a.c.v) +
                                                              spage[j] * a.c.v_stride) +
                              (static_cast<int64_t>(kvh) * a.c.page_size + ((t0 + j) & (a.c.page_size - 1))) * D;
            for (int c = 0; c < C; c++)
                if (tid + 128 * c < D) o[c] = fmaf(sp[j], __half2float(v[tid + 128 * c]), o[c]);
        }
        __syncthreads();
    }
    OutT* out = static_cast<OutT*>(a.out) + (static_cast<int64_t>(b) * a.q_heads + hq) * D;
    for (int c = 0; c < C; c++)
        if (tid + 128 * c < D) out[tid + 128 * c] = from_float<OutT>(l > 0.f ? o[c] / l : 0.f);
    if (a.lse && tid == 0)
        a.lse[static_cast<int64_t>(b) * a.q_heads + hq] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : INFINITY;
}

}  // namespace fp4attn
