// Keys and values into the pages of a cache, quantised as they are written, and back out of it.
//
//   write   bf16:  cache[slot] = x
//           e4m3:  s = max(max_d |x_d|, 1e-8) / 448;  code = e4m3(clamp(x / s, +-448));  scale[slot] = s
//   read    x = bf16(code * s)
//
// The scale belongs to one token of one head, so a row never waits for another one and what is in the cache is never rescaled.
// A NaN or an infinity in a row makes its scale one, and with it everything that is read back of the row.
// Both are bound by memory: 2 D bytes in and D + 4 (or 2 D) bytes out per row, and the other way round.
//
// A lane holds 16 channels of a row (32 bytes of bf16, 16 of codes), the lanes of a row lie side by side (2 .. 16 of them, a
// power of two, so that a row's maximum is a few shuffles), and a thread has kDeep rows in flight.  A block takes a few tokens
// with all their heads, keys and values: what a token needs (its slot; its sequence, page and offset) is looked up once per block.
#include "common.cuh"
#include "kernels.h"

namespace fp8lin {

constexpr int kCacheThreads = 256;
constexpr int kDeep = 4;              // rows that a thread has in flight
constexpr int kMaxTokens = 64;        // tokens of a block

struct CacheGrid {
    int lanes_log2;                   // lanes of a row
    int tokens;                       // tokens of a block
};

// Rows of a block, one behind the other: token, keys then values, head.
struct RowAt {
    int token, head;
    bool values;
};
__device__ __forceinline__ RowAt row_at(int row, int heads) {
    const int token = row / (2 * heads), rest = row - token * 2 * heads;
    const bool values = rest >= heads;
    return {token, values ? rest - heads : rest, values};
}

__device__ __forceinline__ uint32_t max_bits(uint4 w) {
    const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}
// x / s where s is an infinity or a NaN: a zero of x's sign, or a NaN
__device__ __forceinline__ uint2 quant8_not_finite(uint4 w, float s) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = cvt_e4m3x2(__fdiv_rn(bf16_lo(v[i]), s), __fdiv_rn(bf16_hi(v[i]), s));
    return {q[0] | (q[1] << 16), q[2] | (q[3] << 16)};
}

template <bool kE4m3>
__global__ void __launch_bounds__(kCacheThreads)
kv_cache_write_kernel(CacheView c, CacheRows x, const int* slots, CacheGrid grid, int* status) {
    __shared__ int64_t s_at[kMaxTokens], s_scale_at[kMaxTokens];        // where a token lies in the cache, -1: nowhere
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, sub = tid & ((1 << grid.lanes_log2) - 1), lanes_log2 = grid.lanes_log2;
    const int64_t token0 = (int64_t)blockIdx.x * grid.tokens;
    const int tokens = x.rows - token0 < grid.tokens ? (int)(x.rows - token0) : grid.tokens;
    const int rows = tokens * 2 * c.kv_heads, step = kCacheThreads >> lanes_log2;
    const bool mine = sub * 16 < c.dim;
    if (tid < tokens) {
        const int slot = ld_dep(slots + token0 + tid);
        const int64_t page = slot / c.block_size, off = slot - page * c.block_size;
        const bool there = slot >= 0 && page < c.num_blocks;
        if (slot >= 0 && !there) report_status(status, kDevBadPage);
        s_at[tid] = there ? page * c.sb + off * c.st : -1;
        s_scale_at[tid] = page * c.ssb + off * c.sst;
    }
    for (int turn = 0; turn < rows; turn += step * kDeep) {             // (as many for every thread: a row's lanes meet below)
        uint4 w[kDeep][2];
        RowAt at[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            const int row = turn + (tid >> lanes_log2) + i * step;
            at[i] = row_at(row, c.kv_heads);
            w[i][0] = w[i][1] = {0, 0, 0, 0};
            if (row < rows && mine) {
                const int64_t t = token0 + at[i].token;
                const uint4* src = reinterpret_cast<const uint4*>(at[i].values ? x.v + t * x.vt + at[i].head * x.vh : x.k + t * x.kt + at[i].head * x.kh) + 2 * sub;
                w[i][0] = ld_dep(src);
                w[i][1] = ld_dep(src + 1);
            }
        }
        if (turn == 0) __syncthreads();               // the slots, asked for before the rows
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            const int row = turn + (tid >> lanes_log2) + i * step;
            const int64_t to = row < rows ? s_at[at[i].token] : -1;
            unsigned char* dst = (at[i].values ? c.v : c.k) + to + at[i].head * c.sh;
            if (!kE4m3) {
                if (to >= 0 && mine) {
                    reinterpret_cast<uint4*>(dst)[2 * sub] = w[i][0];
                    reinterpret_cast<uint4*>(dst)[2 * sub + 1] = w[i][1];
                }
                continue;
            }
            // |x| as its bits: ordered as the values are, a NaN above the infinity
            uint32_t m = max(max_bits(w[i][0]), max_bits(w[i][1]));
            for (int o = 1; o < 1 << lanes_log2; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (to < 0) continue;
            const float top = __uint_as_float(m << 16), s = __fdiv_rn(m > 0x7f80u ? top : fmaxf(top, 1e-8f), 448.f);
            if (mine) {
                uint2 lo, hi;
                if (m < 0x7f80u) {
                    const ExactDiv div(s);
                    lo = quant8_e4m3(w[i][0], div);
                    hi = quant8_e4m3(w[i][1], div);
                } else {
                    lo = quant8_not_finite(w[i][0], s);
                    hi = quant8_not_finite(w[i][1], s);
                }
                reinterpret_cast<uint4*>(dst)[sub] = {lo.x, lo.y, hi.x, hi.y};
            }
            if (sub == 0) (at[i].values ? c.v_scale : c.k_scale)[s_scale_at[at[i].token] + at[i].head * c.ssh] = s;
        }
    }
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
kv_cache_read_kernel(CacheView c, CacheRows y, const int* tables, int64_t ld_tables, int64_t max_pages, const int* cu, int batch, CacheGrid grid, int* status) {
    __shared__ int64_t s_at[kMaxTokens], s_scale_at[kMaxTokens];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, sub = tid & ((1 << grid.lanes_log2) - 1), lanes_log2 = grid.lanes_log2;
    const int64_t token0 = (int64_t)blockIdx.x * grid.tokens;
    const int tokens = y.rows - token0 < grid.tokens ? (int)(y.rows - token0) : grid.tokens;
    const int rows = tokens * 2 * c.kv_heads, step = kCacheThreads >> lanes_log2;
    if (tid < tokens) {
        const int64_t row = token0 + tid;
        const int b = sequence_of(cu, batch, row);
        int64_t page = -1, off = 0;
        if (b >= 0) {
            const int64_t at = row - ld_dep(cu + b), i = at / c.block_size;
            off = at - i * c.block_size;
            if (i < max_pages) page = ld_dep(tables + b * ld_tables + i);
            if (page < 0 || page >= c.num_blocks) {
                page = -1;
                report_status(status, kDevBadPage);
            }
        }
        s_at[tid] = page < 0 ? -1 : page * c.sb + off * c.st;
        s_scale_at[tid] = page * c.ssb + off * c.sst;
    }
    __syncthreads();
    if (sub * 16 >= c.dim) return;
    for (int row0 = tid >> lanes_log2; row0 < rows; row0 += step * kDeep) {
        uint4 w[kDeep][2];
        float s[kDeep];
        RowAt at[kDeep];
        bool there[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            const int row = row0 + i * step;
            at[i] = row_at(row, c.kv_heads);
            const int64_t from = row < rows ? s_at[at[i].token] : -1;
            there[i] = from >= 0;
            if (there[i]) {
                const uint4* src = reinterpret_cast<const uint4*>((at[i].values ? c.v : c.k) + from + at[i].head * c.sh);
                if (kE4m3) {
                    w[i][0] = ld_dep(src + sub);
                    s[i] = ld_dep((at[i].values ? c.v_scale : c.k_scale) + s_scale_at[at[i].token] + at[i].head * c.ssh);
                } else {
                    w[i][0] = ld_dep(src + 2 * sub);
                    w[i][1] = ld_dep(src + 2 * sub + 1);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            if (!there[i]) continue;
            const int64_t t = token0 + at[i].token;
            uint4* dst = reinterpret_cast<uint4*>(at[i].values ? y.v + t * y.vt + at[i].head * y.vh : y.k + t * y.kt + at[i].head * y.kh) + 2 * sub;
            if (kE4m3) {
                const uint32_t v[4] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w};
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t h = cvt_e4m3x2_to_f16x2((uint16_t)(v[j >> 1] >> (16 * (j & 1))));
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                    o[j] = pack_bf16x2(f.x * s[i], f.y * s[i]);
                }
                dst[0] = {o[0], o[1], o[2], o[3]};
                dst[1] = {o[4], o[5], o[6], o[7]};
            } else {
                dst[0] = w[i][0];
                dst[1] = w[i][1];
            }
        }
    }
}

// Tokens of a block: as many as its threads take in one turn of kDeep rows; fewer where that would leave SMs without a block.
static CacheGrid cache_grid(const CacheView& c, int64_t rows) {
    CacheGrid g = {0, 1};
    while ((16 << g.lanes_log2) < c.dim) ++g.lanes_log2;
    const int at_once = (kCacheThreads >> g.lanes_log2) * kDeep / (2 * c.kv_heads);
    while (g.tokens < kMaxTokens && 2 * g.tokens <= at_once && rows > (int64_t)g.tokens * sm_count()) g.tokens *= 2;
    return g;
}

cudaError_t launch_kv_cache_write(const CacheView& c, const CacheRows& x, const int* slots, int* status, cudaStream_t stream) {
    const CacheGrid g = cache_grid(c, x.rows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((x.rows + g.tokens - 1) / g.tokens));
    cfg.blockDim = dim3(kCacheThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, c.e4m3 ? kv_cache_write_kernel<true> : kv_cache_write_kernel<false>, c, x, slots, g, status));
}

cudaError_t launch_kv_cache_read(const CacheView& c, const CacheRows& y, const int* tables, int64_t ld_tables, int64_t max_pages, const int* cu_seqlens,
                                 int64_t batch, int* status, cudaStream_t stream) {
    const CacheGrid g = cache_grid(c, y.rows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((y.rows + g.tokens - 1) / g.tokens));
    cfg.blockDim = dim3(kCacheThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, c.e4m3 ? kv_cache_read_kernel<true> : kv_cache_read_kernel<false>, c, y, tables, ld_tables, max_pages, cu_seqlens,
                                      (int)batch, g, status));
}

}  // namespace fp8lin
