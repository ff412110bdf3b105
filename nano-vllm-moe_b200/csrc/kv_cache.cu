// Keys and values into the pages of a cache, quantised as they are written, and back out of it.
//
//   write   bf16:  cache[slot] = x
//           e4m3:  s = max(max_d |x_d|, 1e-8) / 448;  code = e4m3(clamp(x / s, +-448));  scale[slot] = s
//   read    x = bf16(code * s)
//
// The scale belongs to one token of one head, so a row never waits for another one and what is in the cache is never rescaled.
// A NaN or an infinity in a row makes its scale one, and with it everything that is read back of the row.
// Both are bound by memory: 2 D bytes in and D + 4 (or 2 D) bytes out per row, and the other way round.
#include "common.cuh"
#include "kernels.h"

namespace fp8lin {

constexpr int kCacheThreads = 256;

// One warp per row (token, keys or values, head); lane i holds the channels 8 i .. 8 i + 7.
template <bool kE4m3>
__global__ void __launch_bounds__(kCacheThreads)
kv_cache_write_kernel(CacheView c, CacheRows x, const int* slots, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5);
    const int64_t token = row / (2 * c.kv_heads);
    if (token >= x.rows) return;
    const int rest = (int)(row - token * (2 * c.kv_heads));
    const bool values = rest >= c.kv_heads;
    const int head = values ? rest - c.kv_heads : rest;
    const int slot = ld_dep(slots + token);
    if (slot < 0) return;
    const int64_t page = slot / c.block_size, off = slot - page * c.block_size;
    if (page >= c.num_blocks) {
        if (lane == 0) report_status(status, kDevBadPage);
        return;
    }
    const __nv_bfloat16* src = values ? x.v + token * x.vt + head * x.vh : x.k + token * x.kt + head * x.kh;
    unsigned char* dst = (values ? c.v : c.k) + page * c.sb + off * c.st + head * c.sh;
    const bool mine = lane * 8 < c.dim;
    uint4 w = {0, 0, 0, 0};
    if (mine) w = ld_dep(reinterpret_cast<const uint4*>(src) + lane);
    if (!kE4m3) {
        if (mine) reinterpret_cast<uint4*>(dst)[lane] = w;
        return;
    }
    // |x| as its bits: ordered as the values are, a NaN above the infinity
    uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    m = max(m & 0xffffu, m >> 16);
    m = __reduce_max_sync(0xffffffffu, m);
    const float s = __fdiv_rn(m > 0x7f80u ? __uint_as_float(m << 16) : fmaxf(__uint_as_float(m << 16), 1e-8f), 448.f);
    if (mine) {
        uint2 codes;
        if (m < 0x7f80u) {
            codes = quant8_e4m3(w, ExactDiv(s));
        } else {                                   // x / inf is a zero of x's sign, everything else a NaN
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = cvt_e4m3x2(__fdiv_rn(bf16_lo(v[i]), s), __fdiv_rn(bf16_hi(v[i]), s));
            codes = {q[0] | (q[1] << 16), q[2] | (q[3] << 16)};
        }
        reinterpret_cast<uint2*>(dst)[lane] = codes;
    }
    if (lane == 0) (values ? c.v_scale : c.k_scale)[page * c.ssb + off * c.sst + head * c.ssh] = s;
}

// The sequence b with cu[b] <= row < cu[b + 1], or -1.
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int64_t row) {
    int lo = 0, hi = batch;                        // cu[lo] <= row < cu[hi], if there is one
    if (row < ld_dep(cu) || row >= ld_dep(cu + batch)) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (ld_dep(cu + mid) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <bool kE4m3>
__global__ void __launch_bounds__(kCacheThreads)
kv_cache_read_kernel(CacheView c, CacheRows y, const int* tables, int64_t ld_tables, int64_t max_pages, const int* cu, int batch, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5);
    const int64_t token = row / (2 * c.kv_heads);
    if (token >= y.rows) return;
    const int rest = (int)(row - token * (2 * c.kv_heads));
    const bool values = rest >= c.kv_heads;
    const int head = values ? rest - c.kv_heads : rest;
    const int b = sequence_of(cu, batch, token);
    if (b < 0) return;
    const int64_t at = token - ld_dep(cu + b), i = at / c.block_size, off = at - i * c.block_size;
    const int64_t page = i < max_pages ? ld_dep(tables + b * ld_tables + i) : -1;
    if (page < 0 || page >= c.num_blocks) {
        if (lane == 0) report_status(status, kDevBadPage);
        return;
    }
    const unsigned char* src = (values ? c.v : c.k) + page * c.sb + off * c.st + head * c.sh;
    __nv_bfloat16* dst = values ? y.v + token * y.vt + head * y.vh : y.k + token * y.kt + head * y.kh;
    if (lane * 8 >= c.dim) return;
    uint4 o;
    if (kE4m3) {
        const float s = ld_dep((values ? c.v_scale : c.k_scale) + page * c.ssb + off * c.sst + head * c.ssh);
        const long long w = ld_dep(reinterpret_cast<const long long*>(src) + lane);
        uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
            const uint32_t h = cvt_e4m3x2_to_f16x2((uint16_t)(w >> (16 * i2)));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            ow[i2] = pack_bf16x2(f.x * s, f.y * s);
        }
    } else {
        o = ld_dep(reinterpret_cast<const uint4*>(src) + lane);
    }
    reinterpret_cast<uint4*>(dst)[lane] = o;
}

cudaError_t launch_kv_cache_write(const CacheView& c, const CacheRows& x, const int* slots, int* status, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((x.rows * 2 * c.kv_heads + kCacheThreads / 32 - 1) / (kCacheThreads / 32)));
    cfg.blockDim = dim3(kCacheThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, c.e4m3 ? kv_cache_write_kernel<true> : kv_cache_write_kernel<false>, c, x, slots, status));
}

cudaError_t launch_kv_cache_read(const CacheView& c, const CacheRows& y, const int* tables, int64_t ld_tables, int64_t max_pages, const int* cu_seqlens,
                                 int64_t batch, int* status, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((y.rows * 2 * c.kv_heads + kCacheThreads / 32 - 1) / (kCacheThreads / 32)));
    cfg.blockDim = dim3(kCacheThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, c.e4m3 ? kv_cache_read_kernel<true> : kv_cache_read_kernel<false>, c, y, tables, ld_tables, max_pages, cu_seqlens,
                                      (int)batch, status));
}

}  // namespace fp8lin
