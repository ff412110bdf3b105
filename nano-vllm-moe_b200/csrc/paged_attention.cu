// Attention of one new token per sequence over the pages of a key-value cache.
//
//   s_i = scale * q . k_i;   o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),   m = max_i s_i
//
// in one pass over the tokens: with every token that raises the maximum, the sums so far are scaled by exp(m_old - m_new).
// One warp per query head, a lane holds eight channels, everything in fp32.
#include "common.cuh"
#include "kernels.h"

namespace fp8lin {

constexpr int kAttnThreads = 128;

template <bool kE4m3>
__device__ __forceinline__ void load_row8(const unsigned char* row, int lane, float s, float (&f)[8]) {
    if (kE4m3) {
        const long long w = ld_dep(reinterpret_cast<const long long*>(row) + lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t h = cvt_e4m3x2_to_f16x2((uint16_t)(w >> (16 * i)));
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
            f[2 * i] = v.x * s;
            f[2 * i + 1] = v.y * s;
        }
    } else {
        const uint4 w = ld_dep(reinterpret_cast<const uint4*>(row) + lane);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = bf16_lo(v[i]); f[2 * i + 1] = bf16_hi(v[i]); }
    }
}

template <bool kE4m3>
__global__ void __launch_bounds__(kAttnThreads)
paged_attention_kernel(AttnArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kAttnThreads / 32) + (threadIdx.x >> 5);
    const int64_t b = row / a.heads;
    if (b >= a.batch) return;
    const int head = (int)(row - b * a.heads);
    const int kvh = head / (a.heads / a.c.kv_heads);
    const bool mine = lane * 8 < a.c.dim;
    float q[8] = {}, o[8] = {}, m = -INFINITY, l = 0.f;
    if (mine) load_row8<false>(reinterpret_cast<const unsigned char*>(a.q + b * a.q_row + head * a.q_head), lane, 1.f, q);
    int len = ld_dep(a.lens + b);
    if ((int64_t)len > a.max_pages * a.c.block_size) {
        len = (int)(a.max_pages * a.c.block_size);
        if (lane == 0) report_status(a.status, kDevBadPage);
    }
    for (int t = 0; t < len; ++t) {
        const int i = t / a.c.block_size, off = t - i * a.c.block_size;
        const int64_t page = ld_dep(a.tables + b * a.ld_tables + i);
        if (page < 0 || page >= a.c.num_blocks) {
            if (lane == 0) report_status(a.status, kDevBadPage);
            continue;
        }
        const int64_t at = page * a.c.sb + off * a.c.st + kvh * a.c.sh, scale_at = page * a.c.ssb + off * a.c.sst + kvh * a.c.ssh;
        float k[8] = {}, v[8] = {}, s = 0.f;
        if (mine) {
            load_row8<kE4m3>(a.c.k + at, lane, kE4m3 ? ld_dep(a.c.k_scale + scale_at) : 1.f, k);
            load_row8<kE4m3>(a.c.v + at, lane, kE4m3 ? ld_dep(a.c.v_scale + scale_at) : 1.f, v);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(q[e], k[e], s);
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.scale;
        const float top = fmaxf(m, s);
        const float old = m == -INFINITY ? 0.f : expf(m - top), p = expf(s - top);
        m = top;
        l = l * old + p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = o[e] * old + p * v[e];
    }
    if (!mine) return;
    const float inv = len > 0 ? 1.f / l : 0.f;
    uint4 w;
    w.x = pack_bf16x2(o[0] * inv, o[1] * inv);
    w.y = pack_bf16x2(o[2] * inv, o[3] * inv);
    w.z = pack_bf16x2(o[4] * inv, o[5] * inv);
    w.w = pack_bf16x2(o[6] * inv, o[7] * inv);
    const int64_t out = b * a.ld_out + (int64_t)head * a.c.dim + lane * 8;
    if (a.out_scale) *reinterpret_cast<uint2*>(static_cast<unsigned char*>(a.out) + out) = quant8_e4m3(w, ExactDiv(fmaxf(ld_dep(a.out_scale), 1e-12f)));
    else *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + out) = w;
}

size_t paged_attention_scratch(int64_t, int64_t, int64_t, bool) { return 0; }

cudaError_t launch_paged_attention(const AttnArgs& a, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((int64_t)a.batch * a.heads + kAttnThreads / 32 - 1) / (kAttnThreads / 32)));
    cfg.blockDim = dim3(kAttnThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, a.c.e4m3 ? paged_attention_kernel<true> : paged_attention_kernel<false>, a));
}

}  // namespace fp8lin
