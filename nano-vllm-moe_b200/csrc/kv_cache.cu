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
// The lanes of a row lie side by side (2 .. 16 of them, a power of two, so that a row's maximum is a few shuffles).  Of bf16 a lane holds two
// words of eight channels, one in either half of the row, so that every load and store of a row's lanes is one stretch; of codes it
// holds 16, even lanes in the row's first half and odd ones in its second, and neighbours exchange half of theirs on the way.
// (Reading 206 MB back took 46 us with a lane's 16 channels side by side on both sides, which writes half sectors, and 50 with two
// times eight codes a lane.)
// A thread has kDeep rows in flight: two of a write, whose rows are two words a lane (to codes: 16384 tokens of 4 heads of 128 13.1 us, with four 14.4; 5000
// tokens 4.8, 6.4; in bf16 it is the other way round where heads leave threads without a row: 6000 tokens of 10 heads of 80 9.1, with four 8.8), four
// of a read (206 MB 37 us, with two 44, with three 39), or one where the call has hardly more for it (few_rows).
// A block takes a few tokens at a time with all their heads, keys and values; what a token needs (its slot; its sequence, page and
// offset) is looked up once, a turn early: looked up when it was needed, it took longer than the rows.
//
// Measured (B200, in a row of calls, inputs larger than L2): writing 51 MB (16384 tokens of 4 heads of 128, to codes) 13.1 us, 17 MB
// of bf16 3.45, 64 tokens 2.1; reading 206 MB of codes back 37 us, 5.5 TB/s, 134 MB of bf16 24 us, 5.6 TB/s, 777 tokens 2.95.  A kernel that only copies 34 MB takes 8.5 us.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace fp8lin {

constexpr int kCacheThreads = 256;
constexpr int kMaxTokens = 64;        // tokens of a block's turn
constexpr int kCacheBlocks = 8;       // blocks of a launch per SM
// Blocks that an SM holds at a time, by the rows that their threads have in flight.
constexpr int held(int deep) { return deep == 1 ? 6 : deep == 2 ? 5 : 4; }
constexpr int kMaxEnds = 1024;        // sequences whose ends fit a block's shared memory

struct CacheGrid {
    int lanes_log2;                   // lanes of a row
    int tokens;                       // tokens of a block's turn
    int turns;                        // of all blocks
    int step_tokens, step_rest;       // a step of a block's threads: whole tokens, rows beside them
    int token_magic;                  // 2^16 / a token's rows, rounded up: row * token_magic / 2^16 is the token of any row below 256
    int blocks;
    Divisor by_page;                  // block_size
};

// Rows of a block, one behind the other: token, keys then values, head.  A thread goes through them in steps of as many as the block takes at a time.
struct RowAt {
    int token, rest;
    __device__ __forceinline__ void step(int tokens, int more, int rows_of_token) {
        token += tokens;
        rest += more;
        if (rest >= rows_of_token) { rest -= rows_of_token; ++token; }
    }
};
// ... and what it reads and writes there: the head's place in the cache and the row outside it, which only moves from token to
// token where a step is one of whole tokens.
struct CacheLane {
    int tid, sub, step, heads, chunks, lanes;
    RowAt at, steps;
    unsigned char* cache;             // of the head, in token 0's place
    float* scales;
    __nv_bfloat16* row;               // outside the cache
    int64_t row_step;                 // a step of `steps.token` tokens, where heads stay
    __device__ __forceinline__ CacheLane(const CacheView& c, const CacheRows& x, const CacheGrid& grid)
        : tid(threadIdx.x), sub(tid & ((1 << grid.lanes_log2) - 1)), step(kCacheThreads >> grid.lanes_log2), heads(c.kv_heads), chunks(c.dim >> 3),
          lanes(1 << grid.lanes_log2), steps{grid.step_tokens, grid.step_rest} {
        const int row = tid >> grid.lanes_log2;
        at.token = row * grid.token_magic >> 16;
        at.rest = row - at.token * 2 * heads;
    }
    __device__ __forceinline__ void place(const CacheView& c, const CacheRows& x, int token0) {
        const bool values = at.rest >= heads;
        const int head = values ? at.rest - heads : at.rest;
        cache = (values ? c.v : c.k) + head * c.sh;
        scales = (values ? c.v_scale : c.k_scale) + head * c.ssh;
        row = (values ? x.v : x.k) + (token0 + at.token) * (values ? x.vt : x.kt) + head * (values ? x.vh : x.kh);
        row_step = steps.token * (values ? x.vt : x.kt);
    }
    __device__ __forceinline__ void next(const CacheView& c, const CacheRows& x, int token0) {
        at.step(steps.token, steps.rest, 2 * heads);
        if (steps.rest == 0) row += row_step;
        else place(c, x, token0);
    }
};

__device__ __forceinline__ uint2 neighbours(uint2 x) { return {__shfl_xor_sync(0xffffffffu, x.x, 1), __shfl_xor_sync(0xffffffffu, x.y, 1)}; }

// The larger magnitudes of two pairs of bf16 numbers (a NaN is the largest); the signs are of no use.
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// x / s for eight values where neither quotients nor what leads to them can overflow: a quotient refined as in ExactDiv, but of -x, whose
// codes are then negated; computed that way zeros keep their signs.  (nr, s: -1 / s and s, twice)
__device__ __forceinline__ uint2 quant8_finite(uint4 v, uint64_t nr, uint64_t s) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t x = pack_f32x2(bf16_lo(w[i]), bf16_hi(w[i]));
        const uint64_t q0 = mul_f32x2(x, nr);
        c[i] = cvt_e4m3x2(fma_f32x2(fma_f32x2(q0, s, x), nr, q0));
    }
    return {(c[0] | (c[1] << 16)) ^ 0x80808080u, (c[2] | (c[3] << 16)) ^ 0x80808080u};
}
// ... and in general; where s is an infinity or a NaN: a zero of x's sign, or a NaN
__device__ __forceinline__ uint2 quant8_any(uint4 w, float s) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = cvt_e4m3x2(__fdiv_rn(bf16_lo(v[i]), s), __fdiv_rn(bf16_hi(v[i]), s));
    return {q[0] | (q[1] << 16), q[2] | (q[3] << 16)};
}

// Where a token lies in the cache: byte offset of its rows, element offset of its scales; -1: nowhere.
struct TokenAt {
    int64_t row, scale;
};
__device__ __forceinline__ TokenAt token_at(const CacheView& c, int64_t page, int64_t off, int* status) {
    if (page < 0 || page >= c.num_blocks) {
        report_status(status, kDevBadPage);
        return {-1, -1};
    }
    return {page * c.sb + off * c.st, page * c.ssb + off * c.sst};
}

template <bool kE4m3, int kDeep>
__global__ void __launch_bounds__(kCacheThreads, held(kDeep))
kv_cache_write_kernel(CacheView c, CacheRows x, const int* slots, CacheGrid grid, int* status) {
    __shared__ TokenAt s_at[2][kMaxTokens];
    pdl_launch_dependents();
    const CacheLane origin(c, x, grid);
    const int word0 = origin.sub, word1 = origin.sub + origin.lanes;     // of eight bf16 channels
    const bool low = word0 < origin.chunks, high = word1 < origin.chunks, odd = origin.sub & 1;
    const int code = (origin.sub >> 1) + (odd ? origin.lanes >> 1 : 0);  // of 16 codes
    pdl_wait();
    auto tokens_of = [&](int turn) {
        const int left = (int)x.rows - turn * grid.tokens;
        return left < grid.tokens ? left : grid.tokens;
    };
    auto slot_of = [&](int turn) { return turn < grid.turns && origin.tid < tokens_of(turn) ? ld_dep(slots + turn * grid.tokens + origin.tid) : -1; };
    auto put = [&](int slot, int side) {
        if (origin.tid >= kMaxTokens) return;
        const int page = grid.by_page.quotient(slot);
        s_at[side][origin.tid] = slot < 0 ? TokenAt{-1, -1} : token_at(c, page, slot - page * c.block_size, status);
    };
    int slot = slot_of(blockIdx.x), side = 0;
    bool placed = false;
    for (int turn = blockIdx.x; turn < grid.turns; turn += gridDim.x, side ^= 1) {
        const int token0 = turn * grid.tokens;
        const int tokens = tokens_of(turn), rows = tokens * 2 * c.kv_heads;
        CacheLane me = origin;
        me.place(c, x, token0);
        for (int row0 = 0; row0 < rows; row0 += me.step * kDeep) {       // (as often for every thread: a row's lanes meet below)
            uint4 w[kDeep][2];
            CacheLane it = me;
#pragma unroll
            for (int i = 0; i < kDeep; ++i, it.next(c, x, token0)) {
                w[i][0] = w[i][1] = {0, 0, 0, 0};
                if (it.at.token < tokens) {
                    const uint4* src = reinterpret_cast<const uint4*>(it.row);
                    if (low) w[i][0] = ld_dep(src + word0);
                    if (high) w[i][1] = ld_dep(src + word1);
                }
            }
            if (!placed) {                                               // the first slots, asked for in front of the rows
                put(slot, side);
                placed = true;
                __syncthreads();
            }
            if (row0 == 0) slot = slot_of(turn + gridDim.x);
#pragma unroll
            for (int i = 0; i < kDeep; ++i, me.next(c, x, token0)) {
                const TokenAt to = me.at.token < tokens ? s_at[side][me.at.token] : TokenAt{-1, -1};
                unsigned char* dst = me.cache + to.row;
                if (!kE4m3) {
                    if (to.row >= 0 && low) reinterpret_cast<uint4*>(dst)[word0] = w[i][0];
                    if (to.row >= 0 && high) reinterpret_cast<uint4*>(dst)[word1] = w[i][1];
                    continue;
                }
                // |x| as its bits: ordered as the values are, a NaN above the infinity
                const uint4 &a = w[i][0], &b = w[i][1];
                const uint32_t m2 = max_abs2(max_abs2(max_abs2(a.x, a.y), max_abs2(a.z, a.w)), max_abs2(max_abs2(b.x, b.y), max_abs2(b.z, b.w)));
                uint32_t m = max(m2 & 0x7fffu, (m2 >> 16) & 0x7fffu);
                for (int o = 1; o < me.lanes; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                // top / 448, correctly rounded as in ExactDiv (where top is not finite, the first product is the answer)
                const float top = m > 0x7f80u ? __uint_as_float(m << 16) : fmaxf(__uint_as_float(m << 16), 1e-8f), r448 = 1.f / 448.f, q0 = top * r448;
                const float s = m < 0x7f80u ? fmaf(fmaf(-q0, 448.f, top), r448, q0) : q0;
                uint2 c0, c1;
                if (top < 1e38f) {                                      // quotients are 448 at most, and what leads to them is no larger than top
                    const float r = __frcp_rn(s);
                    const uint64_t nr = pack_f32x2(-r, -r), ss = pack_f32x2(s, s);
                    c0 = quant8_finite(a, nr, ss);
                    c1 = quant8_finite(b, nr, ss);
                } else {
                    c0 = quant8_any(a, s);
                    c1 = quant8_any(b, s);
                }
                const uint2 got = neighbours(odd ? c0 : c1);
                if (to.row >= 0) {
                    if (code * 2 < me.chunks) reinterpret_cast<uint4*>(dst)[code] = odd ? uint4{got.x, got.y, c1.x, c1.y} : uint4{c0.x, c0.y, got.x, got.y};
                    if (me.sub == 0) me.scales[to.scale] = s;
                }
            }
        }
        if (turn + gridDim.x >= grid.turns) break;
        put(slot, side ^ 1);
        __syncthreads();
    }
}

// The sequence b with cu[b] <= row < cu[b + 1], or -1.
template <class Ends>
__device__ __forceinline__ int sequence_of(Ends cu, int batch, int row) {
    int lo = 0, hi = batch;                        // cu[lo] <= row < cu[hi], if there is one
    if (row < cu(0) || row >= cu(batch)) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu(mid) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <bool kE4m3, int kDeep>
__global__ void __launch_bounds__(kCacheThreads, held(kDeep))
kv_cache_read_kernel(CacheView c, CacheRows y, const int* tables, int64_t ld_tables, int64_t max_pages, const int* cu, int batch, CacheGrid grid, int* status) {
    __shared__ TokenAt s_at[2][kMaxTokens];
    __shared__ int s_ends[kMaxEnds + 1];
    pdl_launch_dependents();
    const CacheLane origin(c, y, grid);
    const int tid = origin.tid;
    const int word0 = origin.sub, word1 = origin.sub + origin.lanes;     // of eight bf16 channels
    const bool low = word0 < origin.chunks, high = word1 < origin.chunks, odd = origin.sub & 1;
    const int code = (origin.sub >> 1) + (odd ? origin.lanes >> 1 : 0);  // of 16 codes
    pdl_wait();
    if (batch <= kMaxEnds)
        for (int i = tid; i <= batch; i += kCacheThreads) s_ends[i] = ld_dep(cu + i);
    __syncthreads();
    // A token's page and offset; the page on its way.
    struct Looked { int off, page; bool there; };
    auto look = [&](int turn) {
        Looked l = {0, -1, false};
        const int row = turn * grid.tokens + tid;
        if (turn >= grid.turns || tid >= grid.tokens || row >= (int)y.rows) return l;
        int b, from = 0;
        if (batch <= kMaxEnds) {
            b = sequence_of([&](int i) { return s_ends[i]; }, batch, row);
            if (b >= 0) from = s_ends[b];
        } else {
            b = sequence_of([&](int i) { return ld_dep(cu + i); }, batch, row);
            if (b >= 0) from = ld_dep(cu + b);
        }
        if (b < 0) return l;
        l.there = true;
        const int at = (int)((uint32_t)row - (uint32_t)from);
        if (at < 0) return l;                                            // (only where a sequence begins below 0: no page)
        const int i = grid.by_page.quotient(at);
        l.off = at - i * c.block_size;
        if (i < max_pages) l.page = ld_dep(tables + b * ld_tables + i);
        return l;
    };
    auto put = [&](const Looked& l, int side) {
        if (tid < kMaxTokens) s_at[side][tid] = l.there ? token_at(c, l.page, l.off, status) : TokenAt{-1, -1};
    };
    int side = 0;
    put(look(blockIdx.x), side);
    __syncthreads();
    for (int turn = blockIdx.x; turn < grid.turns; turn += gridDim.x, side ^= 1) {
        const int token0 = turn * grid.tokens;
        const int tokens = y.rows - token0 < grid.tokens ? (int)(y.rows - token0) : grid.tokens;
        const Looked next = look(turn + gridDim.x);
        CacheLane me = origin;
        me.place(c, y, token0);
        for (int row0 = 0; row0 < tokens * 2 * c.kv_heads; row0 += me.step * kDeep) {      // (as often for every thread: neighbours meet below)
            uint4 w[kDeep][2] = {};
            float s[kDeep] = {};
            CacheLane it = me;
            bool there[kDeep];
#pragma unroll
            for (int i = 0; i < kDeep; ++i, it.next(c, y, token0)) {
                const TokenAt from = it.at.token < tokens ? s_at[side][it.at.token] : TokenAt{-1, -1};
                there[i] = from.row >= 0;
                if (there[i]) {
                    const unsigned char* src = it.cache + from.row;
                    if (kE4m3) {
                        if (code * 2 < it.chunks) w[i][0] = ld_dep(reinterpret_cast<const uint4*>(src) + code);
                        s[i] = ld_dep(it.scales + from.scale);
                    } else {
                        if (low) w[i][0] = ld_dep(reinterpret_cast<const uint4*>(src) + word0);
                        if (high) w[i][1] = ld_dep(reinterpret_cast<const uint4*>(src) + word1);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kDeep; ++i, me.next(c, y, token0)) {
                uint4* dst = reinterpret_cast<uint4*>(me.row);
                if (kE4m3) {
                    const uint64_t ss = pack_f32x2(s[i], s[i]);
                    auto widened = [&](uint32_t x, uint32_t z) {         // eight codes
                        uint32_t o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t h = cvt_e4m3x2_to_f16x2((uint16_t)((j < 2 ? x : z) >> (16 * (j & 1))));
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                            float lo, hi;
                            unpack_f32x2(mul_f32x2(pack_f32x2(f.x, f.y), ss), lo, hi);
                            o[j] = pack_bf16x2(lo, hi);
                        }
                        return uint4{o[0], o[1], o[2], o[3]};
                    };
                    const uint2 c0 = {w[i][0].x, w[i][0].y}, c1 = {w[i][0].z, w[i][0].w}, got = neighbours(odd ? c0 : c1);
                    if (there[i] && low) dst[word0] = odd ? widened(got.x, got.y) : widened(c0.x, c0.y);
                    if (there[i] && high) dst[word1] = odd ? widened(c1.x, c1.y) : widened(got.x, got.y);
                } else if (there[i]) {
                    if (low) dst[word0] = w[i][0];
                    if (high) dst[word1] = w[i][1];
                }
            }
        }
        if (turn + gridDim.x >= grid.turns) break;
        put(next, side ^ 1);
        __syncthreads();
    }
}

static int lanes_log2(int dim) {
    int l = 1;
    while ((16 << l) < dim) ++l;
    return l;
}

// Tokens of a block's turn: an SM's share where that is less than what a block's threads take at once, `deep` rows each.  Else that many, or
// the power of two below, or twice as many where all blocks that the chip holds still get a turn, whichever leaves the SM with the most turns
// the least to do.  A turn costs, in terms of the bytes of what the threads take at once, those of its tokens, one for each step of its threads and
// a quarter beside them.  (Reading up to 1404 tokens of 10 heads of 80 for 11 sequences: 6 or 12 tokens 15.6 us, the power of two 18.1; 206 MB of 4
// heads of 128: 32 tokens 37.0, 16 tokens 38.2; writing 5000 tokens of 4 heads of 128 to codes: 8 tokens 4.8, 16, too few for the chip's blocks, 6.6;
// 50000 tokens: 16 tokens 32.9, 8 tokens 37.0.)
static CacheGrid cache_grid(const CacheView& c, int64_t rows, int deep) {
    CacheGrid g = {};
    g.lanes_log2 = lanes_log2(c.dim);
    g.tokens = 1;
    const int step = kCacheThreads >> g.lanes_log2, rows_of_token = 2 * c.kv_heads;
    g.step_tokens = step / rows_of_token;
    g.step_rest = step % rows_of_token;
    g.token_magic = 65536 / rows_of_token + 1;
    g.by_page = Divisor(c.block_size);
    const int at_once = std::min(step * deep / rows_of_token, kMaxTokens);
    const int64_t sms = sm_count(), spread = (rows + sms - 1) / sms;
    if (spread <= at_once) {
        g.tokens = (int)spread;
    } else if (at_once > 1) {
        int64_t least = INT64_MAX;
        auto consider = [&](int tokens, int steps) {
            const int64_t cost = ((rows + tokens * sms - 1) / (tokens * sms)) * (4 * tokens + (4 * steps + 1) * at_once);
            if (tokens > kMaxTokens || cost > least) return;
            least = cost;
            g.tokens = tokens;
        };
        int power = 1;
        while (2 * power <= at_once) power *= 2;
        consider(power, 1);
        consider(at_once, 1);
        if (rows >= 2 * at_once * sms * held(deep)) consider(2 * at_once, 2);
    }
    g.turns = (int)((rows + g.tokens - 1) / g.tokens);
    const int64_t most = kCacheBlocks * sms;
    g.blocks = (int)(g.turns < most ? g.turns : most);
    return g;
}

// Whether a row a thread is the better way: while blocks of as many tokens as their threads take at once, a row each, are at most `most` per SM; in bf16,
// where a row costs little beside a block's start, at most 3 if more than a tenth of the threads has no row (10 heads of 80: 12 of 32).  Measured, one row
// against several:
// writes, 7: 937 tokens of 16 heads of 128 to codes 4.5 us and 4.65, 1184 tokens 5.0 and 4.3; 4000 of 3 heads 4.3 and 5.5, 6000 5.8 and 5.7; bf16
// 4000 of 3 heads 3.3 and 3.4, 6000 4.3 and 3.6, 150 of 10 heads of 80 1.9 and 2.1, 600 3.0 and 2.6, 1500 5.15 and 3.3;
// reads, 8: 17 sequences of 276 to 552 tokens of 2 heads of 128 from codes 4.3 and 5.3, 36 of up to 438 tokens of 4 heads 7.7 and 6.1; 900 tokens of 10 heads of
// 80 5.3 and 5.7, 1700 7.75 and 6.2; bf16 4000 of 3 heads of 128 3.8 and 4.3, 6000 5.1 and 4.9, 150 of 10 heads of 80 2.4 and 2.8, 740 3.6 and 3.2.
static bool few_rows(const CacheView& c, int64_t tokens, int most) {
    const int step = kCacheThreads >> lanes_log2(c.dim), rows_of_token = 2 * c.kv_heads, at_once = step / rows_of_token;
    const int64_t blocks = at_once ? (tokens + at_once - 1) / at_once : (tokens * rows_of_token + step - 1) / step;
    const int used = at_once ? at_once * rows_of_token : rows_of_token, of = at_once ? step : (rows_of_token + step - 1) / step * step;
    return blocks <= (int64_t)sm_count() * (c.e4m3 || used * 10ll >= of * 9ll ? most : 3);
}

template <class Kernel, class... Args>
static cudaError_t launch_cache(Kernel kernel, int blocks, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kCacheThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, kernel, args...));
}

cudaError_t launch_kv_cache_write(const CacheView& c, const CacheRows& x, const int* slots, int* status, cudaStream_t stream) {
    const bool few = few_rows(c, x.rows, 7);
    const CacheGrid g = cache_grid(c, x.rows, few ? 1 : 2);
    auto kernel = c.e4m3 ? (few ? kv_cache_write_kernel<true, 1> : kv_cache_write_kernel<true, 2>)
                         : (few ? kv_cache_write_kernel<false, 1> : kv_cache_write_kernel<false, 2>);
    return launch_cache(kernel, g.blocks, stream, c, x, slots, g, status);
}

cudaError_t launch_kv_cache_read(const CacheView& c, const CacheRows& y, const int* tables, int64_t ld_tables, int64_t max_pages, const int* cu_seqlens,
                                 int64_t batch, int* status, cudaStream_t stream) {
    const bool few = few_rows(c, y.rows, 8);
    const CacheGrid g = cache_grid(c, y.rows, few ? 1 : 4);
    auto kernel = c.e4m3 ? (few ? kv_cache_read_kernel<true, 1> : kv_cache_read_kernel<true, 4>)
                         : (few ? kv_cache_read_kernel<false, 1> : kv_cache_read_kernel<false, 4>);
    return launch_cache(kernel, g.blocks, stream, c, y, tables, ld_tables, max_pages, cu_seqlens, (int)batch, g, status);
}

}  // namespace fp8lin
