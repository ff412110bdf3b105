// Attention of one new token per sequence over the pages of a key-value cache.
//
//   s_i = scale * q . k_i;   o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),   m = max_i s_i
//
// in one pass over the tokens: where a block of them exceeds the reference m by 2^8, the sums so far are scaled to a new one.
// What bounds it is the cache's bytes: 2 D of them (bf16: 4 D) per token and key head, against 4 D multiplications for each of the group of
// query heads that share it.  Each byte is read once for up to 8 or 16 query heads on a key head; a larger group is cut into parts that read it
// once each (60 sequences of 100 to 3000 tokens, 20 heads on one of 128, e4m3, three parts: 25 us; at one byte once, the bytes take 4).
//
// Work.  The cached tokens of a key head are cut into tiles of 16 or 32; a query group ("segment": one sequence, one key head, up to
// 8 or 16 of its query heads) is a run of tiles, and all segments one behind the other are one list.  CTAs (one per SM) take
// shares of the list, their warps equal shares of that, so a batch of any lengths keeps every SM busy to the end, and a
// captured call follows lengths that change: the shares are computed on the device, by every warp for itself, from the
// lengths alone.  A segment that several warps share is joined in the CTA; one that several CTAs share by the CTA that
// comes last, over the pieces in the order of the list (so that the result does not depend on which one comes last).
//
// A warp works alone on its tiles: it copies keys and values into a ring of its own with cp.async (16 bytes a lane, rows of any
// stride, zeros for what lies behind the end), several tiles ahead, and never meets a CTA barrier on the way.
//
// Products.  S^T = K Q^T and O^T += V^T P^T with mma.sync.m16n8k16: the tokens, then the channels are the 16 rows, the query heads
// the 8 columns, so that a group of up to 8 costs half the instructions that queries as rows would, and both products' sums
// lie with the same columns in the same lanes.  (tcgen05 would take the tiles as they are, but the tensor cores are busy 10 to 20% of
// the cycles here, and its sums would have to go through tensor memory to meet the softmax.)
// P is split into two numbers of 16 bits, so the weights are good to 2^-16 (bf16) or 2^-21 (f16) instead of 2^-8, for a third
// of the matrix instructions and 1% of the time.
// e4m3 codes are widened to f16 (exact) behind ldmatrix.  Queries are scaled by a power of two into f16's range; a token's
// key scale multiplies its scores, its value scale its weight.  That product is what has to fit f16: per query head it is relative to
// a power of two near the largest product so far, wherever the largest score and the largest scale are, so a token's part of the
// result is off by 2^-21 of itself or 2^-31 of the largest product of a weight and 448 of its row's value scale.  (Weights below 2^-126 of the largest are none;
// scales below 2^kLeast lose digits.  Relative to the largest scale alone it took 256 sequences of up to 512 tokens 13.35 us instead of
// 13.55, a group of 12 heads 31.0 instead of 32.0, the long and the full batches the same, and lost what a quiet token gave beside a louder value.)
//
// Measured (B200, in a row of calls, inputs larger than L2): 311 MB of an e4m3 cache (64 sequences of 1000 to 8192 tokens, 28 heads on 4 of 128) 62 us,
// 5.0 TB/s; 282 MB of a bf16 one (32 sequences of 100 to 2048, 16 heads on 16) 56 us, 5.0 TB/s; 138 MB (one sequence of 131071, e4m3) 35 us,
// 4.0 TB/s; one sequence of 17 tokens 5.1 us.  A kernel that only copies the same bytes in the same way takes 49, 44 and 25 us.  The rest
// is 2.5 us to the first copy (lengths, shares, table), 5 us from the last tile to the result (joining in the CTA and over CTAs, mostly instructions
// that are fetched for the first time), and the SMs' unequal distance from memory.
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace fp8lin {
namespace {

constexpr int kBlock = 16;                      // tokens of a matrix instruction
constexpr int kMaxCtas = 192;                   // of a launch: one per SM
constexpr int kJoin = 16;                       // pieces that a CTA joins at a time
static_assert(3 * kMaxCtas <= kWsMaxCounters, "counters: two per CTA for its pieces, one for a segment's second step");
constexpr float kLog2e = 1.4426950408889634f;

template <bool kE4m3_, int kD_, int kN_, int kM_, int kWarps_, int kStages_>
struct Shape {
    static constexpr bool kE4m3 = kE4m3_;
    static constexpr int kD = kD_;              // channels in shared memory: head_dim rounded up, zeros behind it
    static constexpr int kN = kN_;              // groups of 8 query heads
    static constexpr int kHeads = 8 * kN;
    static constexpr int kM = kM_;              // blocks of 16 tokens in a tile
    static constexpr int kTile = kBlock * kM;
    static constexpr int kWarps = kWarps_;
    static constexpr int kStages = kStages_;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kJoinTiles = 8 / (kM * kN);                      // tiles that take a warp as long as a CTA's joining of a segment that others work on too
    static constexpr int kRow = kD * (kE4m3 ? 1 : 2);                     // bytes of a row
    static constexpr int kWords = kRow / 16;                              // 16-byte words of a row
    static constexpr int kRowsPerCopy = kWords >= 32 ? 1 : 32 / kWords;   // rows that a warp's copy instruction takes
    static constexpr int kCopies = kBlock / kRowsPerCopy;
    static constexpr int kStageBytes = 2 * kTile * kRow + (kE4m3 ? 2 * kTile * 4 : 0);
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kPiece = kHeads * kD;                            // floats of a piece's sums
    static_assert(kPiece * 4 <= kStages * kStageBytes, "a warp's sums lie in its ring");
    static_assert(kWords <= 32, "a row is one copy instruction of a warp at most");
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {              // of an 8 x 8 matrix of 16-bit numbers
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool kF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (kF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Places in the list that a segment takes beside its tiles: beginning and ending one of a single tile takes a warp twice as long as the tile.
constexpr int kBegin = 1;
// The reference of no score at all; exp2(kNone - m) is 0 for that of any.
constexpr float kNone = -3.402823466e38f;
// Weights are relative to a score that is at most 2^kSlack below the largest: it follows the maximum only where that
// runs away from it, so that the sums are rescaled once or twice per segment and not with every new maximum.
constexpr float kSlack = 8.f;
// e4m3: the same for weights times value scales, in f16: 2^kTop for the largest that a reference was made of, 2^(kTop + kSlack) at most.
constexpr float kTop = 6.f;
// Smaller value scales (the formula's are 2^-36 at least) count as this one where references are made.
constexpr float kLeast = -100.f;
__device__ __forceinline__ float log2_approx(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float power_of_2(int e) { return __int_as_float((e + 127) << 23); }                     // e from -126 to 127
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }                 // of a positive number
__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Four e4m3 codes to f16: the lower two, the upper two.
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = cvt_e4m3x2_to_f16x2((uint16_t)w);
    hi = cvt_e4m3x2_to_f16x2((uint16_t)(w >> 16));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t sel) { return __byte_perm(a, 0, sel); }

// Two numbers as hi + lo, each of 16 bits.
template <bool kF16>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    if (kF16) {
        hi = pack_f16x2(x, y);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        lo = pack_f16x2(x - f.x, y - f.y);
    } else {
        hi = pack_bf16x2(x, y);
        lo = pack_bf16x2(x - bf16_lo(hi), y - bf16_hi(hi));
    }
}

// Adds one: what this block wrote before is there for whoever sees the sum, and what others wrote before theirs for this block.
__device__ __forceinline__ int arrive(int* counter) {
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    return old;
}

// Tiles of a sequence; an empty one has one as well, of nothing, so that its zeros are written like any result.
__device__ __forceinline__ int within(int len, int64_t most) { return len < 0 ? 0 : (int64_t)len > most ? (int)most : len; }
__device__ __forceinline__ int tokens_of(const AttnArgs& a, int64_t b, int64_t most) { return within(ld_dep(a.lens + b), most); }
template <int kTile>
__device__ __forceinline__ int tiles_in(int len) { return len > kTile ? (int)(((unsigned)len + kTile - 1) / kTile) : 1; }

// (a division of 64 bits is a hundred instructions, on the way of every call)
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
    return ((n | d) >> 32) == 0 ? (int64_t)((uint32_t)n / (uint32_t)d) : n / d;
}
struct Piece {                  // part of a segment
    int64_t tile0;              // the place of the segment's first tile, -1: none
    int tiles, b, head0, heads; // its tiles, sequence and query heads
};

// Where results go: bf16, or the codes of the bf16 value.
struct Result {
    const AttnArgs& a;
    const ExactDiv div;
    __device__ __forceinline__ explicit Result(const AttnArgs& args) : a(args), div(args.out_scale ? fmaxf(ld_dep(args.out_scale), 1e-12f) : 1.f) {}
    // two channels of a query head, from element `at` of the result on
    template <bool kCodes>
    __device__ __forceinline__ void put(int64_t at, uint32_t w) const {
        if (kCodes) *reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(a.out) + at) = cvt_e4m3x2(div(bf16_lo(w)), div(bf16_hi(w)));
        else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + at) = w;
    }
    // kCount fragments of the sums O^T, of 16 channels each from c * 16 on, and of query heads n * 8 + 2 t4 (x, z) and
    // n * 8 + 2 t4 + 1 (y, w), times those heads' `inv`.  All lanes of a warp together.
    template <bool kE4m3, bool kCodes, int kCount, class Fragment>
    __device__ __forceinline__ void store(int b, int head0, int heads, int c, int n, Fragment fragment, float2 inv) const {
        const int g = (threadIdx.x & 31) >> 2, t4 = threadIdx.x & 3, dim = a.c.dim;
        const int col = n * 8 + (kE4m3 ? 2 * t4 : g);
        // e4m3: rows g and g + 8 of a fragment are channels 2g and 2g + 1; bf16: g and g + 8, and transposed a lane has two of head g
        const int64_t at = (int64_t)b * a.ld_out + (int64_t)(head0 + col) * dim + c * 16 + 2 * (kE4m3 ? g : t4);
        const bool first = col < heads, second = kE4m3 ? col + 1 < heads : first;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if ((c + i) * 16 >= dim) break;
            const float4 v = fragment(i);
            uint32_t x, y;
            if (kE4m3) {
                x = pack_bf16x2(v.x * inv.x, v.z * inv.x);
                y = pack_bf16x2(v.y * inv.y, v.w * inv.y);
            } else {
                x = transposed(pack_bf16x2(v.x * inv.x, v.y * inv.y));
                y = transposed(pack_bf16x2(v.z * inv.x, v.w * inv.y));
            }
            if (first) put<kCodes>(at + i * 16, x);
            if (second) put<kCodes>(at + i * 16 + (kE4m3 ? dim : 8), y);
        }
    }
    template <bool kE4m3, int kCount, class Fragment>
    __device__ __forceinline__ void store(int b, int head0, int heads, int c, int n, Fragment fragment, float2 inv) const {
        if (a.out_scale) store<kE4m3, true, kCount>(b, head0, heads, c, n, fragment, inv);
        else store<kE4m3, false, kCount>(b, head0, heads, c, n, fragment, inv);
    }
};

// Scratch: the sums of a warp's first piece where it went on to another segment, then two pieces per CTA with their statistics.
template <class S>
__host__ __device__ constexpr size_t scratch_floats(int ctas) {
    return (size_t)ctas * S::kWarps * S::kPiece + (size_t)ctas * 2 * (S::kPiece + 2 * S::kHeads);
}

template <class S>
__global__ void __launch_bounds__(S::kThreads, 1)
paged_attention_kernel(AttnArgs a, int group, int parts) {
    constexpr bool kE4m3 = S::kE4m3;
    constexpr int kTile = S::kTile, kM = S::kM, kJoinTiles = S::kJoinTiles, kD = S::kD, kN = S::kN, kHeads = S::kHeads;
    constexpr int kWarps = S::kWarps, kStages = S::kStages, kRow = S::kRow, kPiece = S::kPiece;
    extern __shared__ __align__(1024) unsigned char ring[];
    __shared__ Piece s_piece[2 * kWarps];
    // (read two heads at a time)
    __shared__ __align__(16) float s_m[2 * kWarps][kHeads], s_l[2 * kWarps][kHeads], s_f[2 * kWarps][kHeads], s_top[kHeads], s_sum[kHeads], s_share[kJoin][kHeads];
    __shared__ int s_entry[2 * kWarps];                                          // the pieces that there are, in the order of the list
    __shared__ int s_last[2], s_cta0[2], s_ctas[2], s_first[2], s_again;                     // segments that other CTAs have pieces of; which CTAs

    auto tiles_of = [](int len) { return tiles_in<kTile>(len); };
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int segments = a.c.kv_heads * parts;                                   // per sequence
    const int64_t most64 = a.max_pages * a.c.block_size, most = most64 < 0x7fffff00 ? most64 : 0x7fffff00;

    // ---- shares: every warp for itself, a lane for a stretch of sequences -------------------------------------------
    const int stretch = (a.batch + 31) >> 5, lane_b = lane * stretch;
    int64_t mine = 0;
    int lane_len = 0, lane_most = 0;                                              // of the stretch's last; most tiles
#pragma unroll 8
    for (int i = 0; i < stretch; ++i) {
        if (lane_b + i < a.batch) {
            const int len = ld_dep(a.lens + lane_b + i);
            if (len > most && blockIdx.x == 0) report_status(a.status, kDevBadPage);
            lane_len = len < 0 ? 0 : len < most ? len : (int)most;
            const int tiles = tiles_of(lane_len);
            mine += tiles;
            lane_most = tiles > lane_most ? tiles : lane_most;
        }
    }
    // Sequence b's part of the list: a segment's tiles with kBegin places in front of them, what beginning and ending it takes.
    auto places_of = [&](int len) { return (int64_t)(tiles_of(len) + kBegin) * segments; };
    auto sum_upto = [&](int64_t x) {                                              // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    // The sequence whose part of a list `at` is in, the place in it, the sequence's length.  part_of: a sequence's part by its length; this
    // lane's stretch begins at `before` and has `mine`.
    struct Found { int b, len; int64_t inside; };
    auto find = [&](auto part_of, int64_t before, int64_t mine, int64_t place) {
        Found f;
        f.inside = place - before;
        const int where = __ffs(__ballot_sync(0xffffffffu, f.inside >= 0 && f.inside < mine)) - 1;
        f.inside = __shfl_sync(0xffffffffu, f.inside, where);
        f.b = where;
        f.len = __shfl_sync(0xffffffffu, lane_len, where);
        if (stretch > 1) for (int b0 = where * stretch; b0 < a.batch; b0 += 32) {  // (it is one of the stretch's)
            const int len = b0 + lane < a.batch ? tokens_of(a, b0 + lane, most) : 0;
            const int64_t all = b0 + lane < a.batch ? part_of(len) : 0, upto = sum_upto(all);
            const uint32_t beyond = __ballot_sync(0xffffffffu, upto > f.inside);
            if (beyond) {
                const int w = __ffs(beyond) - 1;
                f.b = b0 + w;
                f.len = __shfl_sync(0xffffffffu, len, w);
                f.inside -= __shfl_sync(0xffffffffu, upto - all, w);
                break;
            }
            f.inside -= __shfl_sync(0xffffffffu, upto, 31);
        }
        return f;
    };
    // Three ways to deal the list out.
    // (1) To CTAs that work on one segment each, some on the same, where no CTA's share grows by more than a sixteenth: joining the pieces of two
    // segments takes a CTA twice as long.  Joining over CTAs costs as much as kJoinTiles per warp, so where there is a CTA for every segment and none is
    // that much longer than an even share, each has one (17 tokens 5.1 us, where four segments shared one CTA 7.5).
    // (2) Segments of a few tiles: in even shares, rounded to whole segments (256 sequences of up to 512 tokens 13.8 us, joined over CTAs 17.6).
    // (3) In even shares.
    const int longest = __reduce_max_sync(0xffffffffu, lane_most), grid = (int)gridDim.x;
    const bool few = a.batch <= grid && a.batch * segments <= grid;
    bool apart = few && longest <= (1 + kJoinTiles) * kWarps;                     // (a share is a tile per warp at least)
    int64_t total = 0, before = 0, share = kWarps, cta0, cta1;                    // this CTA's places: of the list, or (apart) of one segment's part of it
    Found own = {};                                                               // apart: that segment
    int own_segment = 0, own_part = 0, own_parts = 1;                             // ... which of its CTAs this is, and of how many
    if (apart) {
        if ((int)blockIdx.x >= a.batch * segments) return;
        own.b = a.by_segments.quotient(blockIdx.x);
        own_segment = blockIdx.x - own.b * segments;
        own.len = stretch == 1 ? __shfl_sync(0xffffffffu, lane_len, own.b) : tokens_of(a, own.b, most);
        cta0 = kBegin;
        cta1 = kBegin + tiles_of(own.len);
    } else {
        mine = (mine + (int64_t)kBegin * (a.batch - lane_b < 0 ? 0 : a.batch - lane_b < stretch ? a.batch - lane_b : stretch)) * segments;
        const int64_t before_end = sum_upto(mine);
        total = __shfl_sync(0xffffffffu, before_end, 31);
        before = before_end - mine;
        share = quotient(total + grid - 1, grid);
        if (share < kWarps) share = kWarps;
        if (few) {
            const int64_t cta_share = longest <= share + kJoinTiles * kWarps ? longest : share + share / 16;
            auto units_of = [&](int len) { return quotient(tiles_of(len) + cta_share - 1, cta_share) * segments; };      // CTAs of a sequence
            int64_t units = 0;
            if (stretch == 1) units = lane < a.batch ? units_of(lane_len) : 0;
            else for (int i = 0; i < stretch; ++i)
                if (lane_b + i < a.batch) units += units_of(tokens_of(a, lane_b + i, most));
            const int64_t upto = sum_upto(units), all = __shfl_sync(0xffffffffu, upto, 31);
            apart = all <= grid;
            if (apart) {
                if ((int)blockIdx.x >= all) return;
                own = find(units_of, upto - units, units, blockIdx.x);
                own_parts = (int)quotient(tiles_of(own.len) + cta_share - 1, cta_share);
                own_segment = (int)own.inside / own_parts;
                own_part = (int)own.inside - own_segment * own_parts;
                cta0 = kBegin + own_part * cta_share;
                cta1 = kBegin + tiles_of(own.len);
                if (cta1 > cta0 + cta_share) cta1 = cta0 + cta_share;
            }
        }
        if (!apart) {
            cta0 = blockIdx.x * share;
            cta1 = cta0 + share < total ? cta0 + share : total;
            if (cta0 >= total) return;
            if (longest <= kJoinTiles / 4 * kWarps) {                             // ... to the nearer end of a segment
#pragma unroll 1
                for (int side = 0; side < 2; ++side) {
                    const int64_t place = side == 0 ? cta0 : cta1;
                    if (place >= total) break;
                    const Found f = find(places_of, before, mine, place);
                    const int places = tiles_of(f.len) + kBegin, in_segment = (int)(f.inside - quotient(f.inside, places) * places);
                    const int64_t moved = place + (2 * in_segment < places ? -in_segment : places - in_segment);
                    if (side == 0) cta0 = moved;
                    else cta1 = moved;
                }
                if (cta0 >= cta1) return;
            }
        }
    }
    const int64_t warp_share = (cta1 - cta0 + kWarps - 1) / kWarps, begin = cta0 + warp * warp_share;
    const int64_t span64 = cta1 - begin < warp_share ? cta1 - begin : warp_share;
    const int span = span64 < 0 ? 0 : (int)(span64 < 0x3fffffff ? span64 : 0x3fffffff);                  // this warp's places: from `begin` on

    // ---- a warp's tiles -----------------------------------------------------------------------------------------------
    unsigned char* const my_ring = ring + warp * (kStages * S::kStageBytes);
    const uint32_t my_ring_at = smem_addr(my_ring);
    const int row_bytes = a.c.dim * (kE4m3 ? 1 : 2);
    // (the magic number made here: as a parameter of the launch it took 131071 e4m3 tokens 36.2 us instead of 34.5)
    const int page_size = a.c.block_size, page_magic = page_size <= kBlock ? 65536 / page_size + 1 : 0;
    // (of up to 30 tokens, or of less than two pages)
    auto pages_in = [&](int tokens) { return page_size > kBlock ? (tokens >= page_size ? 1 : 0) : tokens * page_magic >> 16; };
    const int g = lane >> 2, t4 = lane & 3;
    if (row_bytes < kRow) {                                         // channels behind head_dim: zeros once, they are never copied to
        for (int i = lane * 16; i < kStages * S::kStageBytes; i += 512) *reinterpret_cast<uint4*>(my_ring + i) = {0, 0, 0, 0};
        __syncwarp();
    }

    struct Place {
        int b, head, part, t, len, tiles, place;                    // sequence, key head, part of its query heads, tile; its place from `begin` on
    } in = {}, at = {};                                             // of the next tile to copy, and to work on
    auto next_segment = [&](Place& x) {                             // whether it is one of the same sequence
        x.place += kBegin;
        if (++x.part < parts) return true;
        x.part = 0;
        if (++x.head < a.c.kv_heads) return true;
        x.head = 0;
        ++x.b;
        return false;
    };
    // Nothing that the loop needs is waited for in it: a load queues behind all the copies that the SM's warps have asked for, some
    // 2.5 us.  So lengths and queries are asked for a segment early, and pages come 32 table entries at a time, a lane each, also
    // early: those from page_base on, the 32 behind them, a sequence's first for its next head, and the next sequence's.
    // (The walk runs ahead of what there is, behind the last tile of the batch into a sequence that does not exist: `entry` tells it.)
    int pages = 0, pages_behind = 0, pages_first = 0, page_base = 0, page_at = 0, page_off = 0;
    int next_len = 0, next_pages = 0, after_len = 0;                // of the sequences behind in.b, behind at.b
    auto entry = [&](int b, int64_t i) { return b < a.batch && i < a.max_pages ? ld_dep(a.tables + (int64_t)b * a.ld_tables + i) : -1; };
    auto look_at = [&](int b) {
        if (b < a.batch) {
            next_len = ld_dep(a.lens + b);
            next_pages = entry(b, lane);
        }
    };
    if (span > 0) {
        Found f = own;
        int segment = own_segment;
        if (!apart) f = find(places_of, before, mine, begin);
        in.b = f.b;
        in.len = f.len;
        in.tiles = tiles_of(in.len);
        if (apart) f.inside = begin;
        else segment = (int)quotient(f.inside, in.tiles + kBegin);
        in.t = (int)(apart ? begin : f.inside - (int64_t)segment * (in.tiles + kBegin)) - kBegin;
        if (in.t < 0) { in.place = -in.t; in.t = 0; }
        in.head = a.by_parts.quotient(segment);
        in.part = segment - in.head * parts;
        at = in;
        page_base = page_at = a.by_page.quotient(in.t * kTile);
        page_off = in.t * kTile - page_at * page_size;
        pages = entry(in.b, page_base + lane);
        pages_behind = entry(in.b, page_base + 32 + lane);
        pages_first = entry(in.b, lane);
        look_at(in.b + 1);
        if (at.b + 1 < a.batch) after_len = ld_dep(a.lens + at.b + 1);
    }
    // copies: lane -> word `word` of the rows copy_row + j * kRowsPerCopy
    const int copy_row = lane / S::kWords, word = lane % S::kWords;
    auto swizzle = [](int r, int w) { return S::kWords >= 8 ? (w & ~7) | ((w ^ r) & 7) : (w ^ (r >> 1)) & 3; };
    const uint32_t copy_dst = copy_row * kRow + swizzle(copy_row, word) * 16;
    const unsigned page_limit = a.c.num_blocks < 0x7fffffff ? (unsigned)a.c.num_blocks : 0x7fffffffu;
    const bool word_there = word * 16 < row_bytes, dense = a.c.st == kRow;
    const int64_t lane_from = copy_row * a.c.st + word * 16, v_less_k = a.c.v - a.c.k;
    const float* const lane_scale = kE4m3 ? (lane < 16 ? a.c.k_scale : a.c.v_scale) + (lane & 15) * a.c.sst : nullptr;
    auto copy_block = [&](uint32_t ks, uint32_t vs, uint32_t scales, int token0) {
        const int rows = in.len - token0;                                         // that exist: at least 16, but at a sequence's end
        auto dst_of = [&](int j) { return j * S::kRowsPerCopy * kRow + (copy_dst ^ (S::kWords >= 8 ? ((j * S::kRowsPerCopy) & 7) * 16 : 0)); };
        if (page_at - page_base >= 32) {
            page_base += 32;
            pages = pages_behind;
            pages_behind = entry(in.b, page_base + 32 + lane);
        }
        const int at_page = page_at - page_base, off16 = page_off, passed = pages_in(off16 + kBlock);
        page_at += passed;
        page_off += kBlock - passed * page_size;
        if (rows >= kBlock && off16 + kBlock <= page_size) {
            const int page = __shfl_sync(0xffffffffu, pages, at_page);
            if ((unsigned)page < page_limit) {                                    // a whole block of a page
                const unsigned char* k_row = a.c.k + page * a.c.sb + off16 * a.c.st + in.head * a.c.sh + lane_from;
                const unsigned char* v_row = k_row + v_less_k;
                if (word_there) {
                    if (dense) {
#pragma unroll
                        for (int j = 0; j < S::kCopies; ++j) {
                            copy16(ks + dst_of(j), k_row + j * S::kRowsPerCopy * kRow);
                            copy16(vs + dst_of(j), v_row + j * S::kRowsPerCopy * kRow);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < S::kCopies; ++j) {
                            copy16(ks + dst_of(j), k_row);
                            copy16(vs + dst_of(j), v_row);
                            k_row += S::kRowsPerCopy * a.c.st;
                            v_row += S::kRowsPerCopy * a.c.st;
                        }
                    }
                }
                if (kE4m3) copy4(scales + lane * 4, lane_scale + page * a.c.ssb + off16 * a.c.sst + in.head * a.c.ssh, true);
                return;
            }
        }
        // a sequence's end, blocks on several pages, pages that do not exist: row by row, zeros where there is none
        const int r16 = lane & 15, row_page = pages_in(off16 + r16), which = at_page + row_page;
        const int page_here = __shfl_sync(0xffffffffu, pages, which), page_there = __shfl_sync(0xffffffffu, pages_behind, which);     // (lane `which` % 32)
        const int64_t p = which < 32 ? page_here : page_there, off = off16 + r16 - row_page * page_size;
        bool there = r16 < rows;
        if (there && (unsigned)p >= page_limit) {
            there = false;
            report_status(a.status, kDevBadPage);
        }
        const long long row_from = there ? p * a.c.sb + off * a.c.st + in.head * a.c.sh : -1;
#pragma unroll 1
        for (int j = 0; j < S::kCopies; ++j) {
            const long long from = __shfl_sync(0xffffffffu, row_from, copy_row + j * S::kRowsPerCopy);
            const bool ok = from >= 0 && word_there;
            const unsigned char* row = ok ? a.c.k + from + word * 16 : a.c.k;
            copy16(ks + dst_of(j), row, ok);
            copy16(vs + dst_of(j), ok ? row + v_less_k : a.c.v, ok);
        }
        if (kE4m3) {
            const float* s = (lane < 16 ? a.c.k_scale : a.c.v_scale) + (there ? p * a.c.ssb + off * a.c.sst + in.head * a.c.ssh : 0);
            copy4(scales + lane * 4, s, there);
        }
    };
    auto copy_tile = [&](int stage) {
        const uint32_t ks = my_ring_at + stage * S::kStageBytes;
#pragma unroll
        for (int h = 0; h < kM; ++h)
            copy_block(ks + h * kBlock * kRow, ks + (kTile + h * kBlock) * kRow, ks + 2 * kTile * kRow + h * 2 * kBlock * 4, in.t * kTile + h * kBlock);
    };
    auto next_tile = [&] {
        ++in.place;
        if (++in.t < in.tiles) return;
        in.t = 0;
        page_at = page_off = 0;
        if (next_segment(in)) {
            if (page_base != 0) {
                page_base = 0;
                pages = pages_first;
                pages_behind = entry(in.b, 32 + lane);
            }
            return;
        }
        in.len = within(next_len, most);
        in.tiles = tiles_of(in.len);
        page_base = 0;
        pages = pages_first = next_pages;
        pages_behind = entry(in.b, 32 + lane);
        look_at(in.b + 1);
    };

    const Result result(a);
    uint32_t q[kD / 16][kN][2];
    float o[kD / 16][kN][4], m[kN][2], l[kN][2], to_score[kN][2];
    // e4m3: sums are those of weights times value scales times v_up, a power of two.  As long as scores are at most `gap` above m and scales at
    // most v_most, no product is more than 2^kSlack times its reference, whichever score goes with whichever scale.
    float v_up[kN][2], gap = kSlack, v_most = 0.f;
    // Queries are asked for one segment early where registers allow: they queue behind the tiles that the SM's warps have asked for.
    constexpr bool kQueriesEarly = kN == 1 && kD <= 128;
    uint32_t q_next[kQueriesEarly ? kD / 16 : 1][kN][2];
    auto load_queries = [&](uint32_t (&to)[kD / 16][kN][2], const Place& x) {
        const int head0 = x.head * group + x.part * kHeads, heads = group - x.part * kHeads;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const __nv_bfloat16* row = a.q + (int64_t)x.b * a.q_row + (int64_t)(head0 + n * 8 + g) * a.q_head;
            const bool real = n * 8 + g < heads;
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) {
                to[s][n][0] = to[s][n][1] = 0;
                if (real && s * 16 < a.c.dim) {
                    if (kE4m3) {
                        const long long w = ld_dep(reinterpret_cast<const long long*>(row + s * 16 + t4 * 4));
                        to[s][n][0] = (uint32_t)w;
                        to[s][n][1] = (uint32_t)(w >> 32);
                    } else {
                        to[s][n][0] = ld_dep(reinterpret_cast<const int*>(row + s * 16 + t4 * 2));
                        to[s][n][1] = ld_dep(reinterpret_cast<const int*>(row + s * 16 + 8 + t4 * 2));
                    }
                }
            }
        }
    };
    auto begin_segment = [&](bool first) {
        v_most = 0.f;
        gap = kSlack;
        if constexpr (kQueriesEarly) {
            if (first) load_queries(q_next, at);
#pragma unroll
            for (int s = 0; s < kD / 16; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) q[s][0][i] = q_next[s][0][i];
            Place next = at;
            if (next_segment(next) || next.b < a.batch) load_queries(q_next, next);
        } else {
            load_queries(q, at);
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const float base = a.scale * kLog2e;
            if (kE4m3) {
                // the largest channel to 2^14 .. 2^15: f16 holds those down to 2^-29 of it with all of bf16's bits
                uint32_t top = 0;
#pragma unroll
                for (int s = 0; s < kD / 16; ++s) top = __vmaxu2(top, __vmaxu2(q[s][n][0] & 0x7fff7fffu, q[s][n][1] & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = (int)(top >> 7), up = e == 255 ? 0 : 14 + 127 - (e == 0 ? 1 : e);       // -113 .. 140: as two factors
                const float up1 = __int_as_float((127 + (up >> 1)) << 23), up2 = __int_as_float((127 + up - (up >> 1)) << 23);
                const float down1 = __int_as_float((127 - (up >> 1)) << 23), down2 = __int_as_float((127 - up + (up >> 1)) << 23);
#pragma unroll
                for (int s = 0; s < kD / 16; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w = q[s][n][i];
                        q[s][n][i] = pack_f16x2(bf16_lo(w) * up1 * up2, bf16_hi(w) * up1 * up2);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) to_score[n][i] = base * __shfl_sync(0xffffffffu, down1, (2 * t4 + i) * 4) * __shfl_sync(0xffffffffu, down2, (2 * t4 + i) * 4);
            } else {
                to_score[n][0] = to_score[n][1] = base;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[n][i] = kNone;
                l[n][i] = 0.f;
                v_up[n][i] = power_of_2((int)(kTop - kLeast));
            }
#pragma unroll
            for (int c = 0; c < kD / 16; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][n][i] = 0.f;
        }
    };

    // ldmatrix: where this lane's row of a matrix is, for the first channels; word w + its is at the same place ^ (w & 7) * 16, + (w & ~7) * 16
    const int mi = lane >> 3, lr = lane & 7, k_r = lr + (mi & 1) * 8, v_r = kE4m3 ? k_r : lr + (mi >> 1) * 8;
    const uint32_t k_lane = k_r * kRow + swizzle(k_r, mi >> 1) * 16, v_lane = v_r * kRow + swizzle(v_r, kE4m3 ? mi >> 1 : mi & 1) * 16;
    auto words_on = [](uint32_t lane_at, int w) { return (lane_at ^ ((w & 7) * 16)) + (w & ~7) * 16; };
    constexpr int kLoads = kD / (kE4m3 ? 32 : 16);                                 // of a block's keys (or values)
    // Values to registers in front of the softmax, where there are registers for them (with 16 warps per CTA they spill: 256 sequences of
    // up to 512 tokens 13.7 us, without 13.55)
    constexpr bool kEarly = kM * kLoads <= 8 && kWarps <= 8;
    auto work_on = [&](int stage) {
        const uint32_t ks = my_ring_at + stage * S::kStageBytes, k_at = ks + k_lane, v_at = ks + kTile * kRow + v_lane;
        auto load_keys = [&](uint32_t (&f)[4], int h, int x) { ldmatrix4(f, words_on(k_at, 2 * x) + h * kBlock * kRow); };
        auto load_values = [&](uint32_t (&f)[4], int h, int x) { ldmatrix4_trans(f, words_on(v_at, 2 * x) + h * kBlock * kRow); };
        // scores: rows of the A operand are tokens; two sums each, so that they do not wait for one another
        float s[kM][kN][4], s2[kM][kN][4];
#pragma unroll
        for (int h = 0; h < kM; ++h)
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][n][i] = s2[h][n][i] = 0.f;
        constexpr int kAhead = kLoads < 8 / kM ? kLoads : 8 / kM;
#pragma unroll
        for (int x0 = 0; x0 < kLoads; x0 += kAhead) {
            uint32_t f[kM][kAhead][4];
#pragma unroll
            for (int x = 0; x < kAhead; ++x)
#pragma unroll
                for (int h = 0; h < kM; ++h) load_keys(f[h][x], h, x0 + x);
#pragma unroll
            for (int x = 0; x < kAhead; ++x)
#pragma unroll
                for (int h = 0; h < kM; ++h) {
                    const uint32_t* y = f[h][x];
                    if (kE4m3) {
                        uint32_t lo[4], hi[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) widen(y[i], lo[i], hi[i]);
#pragma unroll
                        for (int n = 0; n < kN; ++n) {
                            const int c = 2 * (x0 + x);
                            mma<true>(s[h][n], lo[0], lo[1], hi[0], hi[1], q[c][n][0], q[c][n][1]);
                            mma<true>(s2[h][n], lo[2], lo[3], hi[2], hi[3], q[c + 1][n][0], q[c + 1][n][1]);
                        }
                    } else {
#pragma unroll
                        for (int n = 0; n < kN; ++n) mma<false>((x & 1) ? s2[h][n] : s[h][n], y[0], y[1], y[2], y[3], q[x0 + x][n][0], q[x0 + x][n][1]);
                    }
                }
        }
        uint32_t vf[kM][kEarly ? kLoads : 1][4];
        if (kEarly) {
#pragma unroll
            for (int x = 0; x < kLoads; ++x)
#pragma unroll
                for (int h = 0; h < kM; ++h) load_values(vf[h][x], h, x);
        }
        float k_scale[kM][2], v_scale[kM][2];                                      // of tokens g and g + 8
        if (kE4m3) {
            const float* sc = reinterpret_cast<const float*>(my_ring + stage * S::kStageBytes + 2 * kTile * kRow);
#pragma unroll
            for (int h = 0; h < kM; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) { k_scale[h][i] = sc[h * 32 + g + 8 * i]; v_scale[h][i] = sc[h * 32 + 16 + g + 8 * i]; }
        }
        const int rows = at.len - at.t * kTile;
#pragma unroll
        for (int h = 0; h < kM; ++h)
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][n][i] = (s[h][n][i] + s2[h][n][i]) * (kE4m3 ? k_scale[h][i >> 1] * to_score[n][i & 1] : to_score[n][i & 1]);
        if (rows < kTile) {
#pragma unroll
            for (int h = 0; h < kM; ++h)
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (h * kBlock + g + 8 * (i >> 1) >= rows) s[h][n][i] = -INFINITY;
        }
        float top[kN][2];
        bool raised = false;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                top[n][i] = fmaxf(s[0][n][i], s[0][n][2 + i]);
#pragma unroll
                for (int h = 1; h < kM; ++h) top[n][i] = fmaxf(top[n][i], fmaxf(s[h][n][i], s[h][n][2 + i]));
                raised |= top[n][i] > (kE4m3 ? __fadd_rd(m[n][i], gap) : m[n][i] + kSlack);
            }
        float v_top = 0.f;
        if (kE4m3) {
#pragma unroll
            for (int h = 0; h < kM; ++h) v_top = fmaxf(v_top, fmaxf(fabsf(v_scale[h][0]), fabsf(v_scale[h][1])));
            raised |= v_top > v_most;
        }
        if (__any_sync(0xffffffffu, raised)) {
            // (v_most: the tile's, so that a louder one is forgotten when it has passed.  131071 tokens whose value scales vary by a factor of 3 at one standard
            // deviation take 35.0 us, by 16 36.2.)
            float v_log[kM][2], most = 0.f;
            if (kE4m3) {
                const uint32_t e = __reduce_max_sync(0xffffffffu, __float_as_uint(v_top) >> 23);
                v_most = __uint_as_float(e << 23 | 0x7fffffu);
                most = (float)((int)e - 126);
                gap = kSlack;
#pragma unroll
                for (int h = 0; h < kM; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) v_log[h][i] = fmaxf(log2_approx(fabsf(v_scale[h][i])), kLeast);
            }
            auto lanes_max = [](float x) {
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            };
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = fmaxf(m[n][i], lanes_max(top[n][i])), down = m[n][i] - x, f = exp2_approx(down);
                    float fd = f;
                    m[n][i] = x;
                    l[n][i] *= f;
                    if (kE4m3) {
                        float y = -INFINITY;                                       // of the scores' distances from m: scores may be far larger than the scales' logarithms
#pragma unroll
                        for (int h = 0; h < kM; ++h)
#pragma unroll
                            for (int r = 0; r < 2; ++r) y = fmaxf(y, s[h][n][2 * r + i] - x + v_log[h][r]);
                        const float before = kTop - (float)exponent(v_up[n][i]) + down;
                        const float ref = fminf(fmaxf(ceilf(fmaxf(before, lanes_max(y))), kLeast), 129.f);     // (beyond them: infinities and NaN)
                        fd = exp2_approx(before - ref);
                        v_up[n][i] = power_of_2((int)(kTop - ref));
                        gap = fminf(gap, ref + kSlack - most);
                    }
#pragma unroll
                    for (int c = 0; c < kD / 16; ++c) { o[c][n][i] *= fd; o[c][n][2 + i] *= fd; }
                }
        }
        uint32_t hi[kM][kN][2], lo[kM][kN][2];
#pragma unroll
        for (int h = 0; h < kM; ++h) {
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float p[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        p[i] = exp2_approx(s[h][n][2 * r + i] - m[n][i]);
                        l[n][i] += p[i];
                    }
                    if (kE4m3)                                                     // (v_up first: it undoes what a scale far from 1 does)
                        unpack_f32x2(mul_f32x2(mul_f32x2(pack_f32x2(p[0], p[1]), pack_f32x2(v_up[n][0], v_up[n][1])), pack_f32x2(v_scale[h][r], v_scale[h][r])), p[0], p[1]);
                    split2<kE4m3>(p[0], p[1], hi[h][n][r], lo[h][n][r]);
                    hi[h][n][r] = transposed(hi[h][n][r]);
                    lo[h][n][r] = transposed(lo[h][n][r]);
                }
        }
        // values: rows of the A operand are channels
#pragma unroll
        for (int x = 0; x < kLoads; ++x)
#pragma unroll
            for (int h = 0; h < kM; ++h) {
                uint32_t late[4];
                if (!kEarly) load_values(late, h, x);
                const uint32_t* y = kEarly ? vf[h][kEarly ? x : 0] : late;
                if (kE4m3) {
                    // a lane's word holds channels 2g and 2g + 1 of two tokens: the first are row g, the second row g + 8
                    uint32_t even[4], odd[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) widen(prmt(y[i], 0x3120), even[i], odd[i]);
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        mma<true>(o[2 * x][n], even[0], odd[0], even[1], odd[1], hi[h][n][0], hi[h][n][1]);
                        mma<true>(o[2 * x + 1][n], even[2], odd[2], even[3], odd[3], hi[h][n][0], hi[h][n][1]);
                        mma<true>(o[2 * x][n], even[0], odd[0], even[1], odd[1], lo[h][n][0], lo[h][n][1]);
                        mma<true>(o[2 * x + 1][n], even[2], odd[2], even[3], odd[3], lo[h][n][0], lo[h][n][1]);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        mma<false>(o[x][n], y[0], y[1], y[2], y[3], hi[h][n][0], hi[h][n][1]);
                        mma<false>(o[x][n], y[0], y[1], y[2], y[3], lo[h][n][0], lo[h][n][1]);
                    }
                }
            }
    };
    // A piece's sums, as they lie in the lanes, with their statistics; `last`: the warp's last piece, kept in shared memory, else in scratch.
    auto keep_piece = [&](bool last, float* sums) {
        const int e = 2 * warp + last;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            if (g == 0) {
                *reinterpret_cast<float2*>(&s_m[e][n * 8 + 2 * t4]) = {m[n][0], m[n][1]};
                *reinterpret_cast<float2*>(&s_l[e][n * 8 + 2 * t4]) = {l[n][0], l[n][1]};
            }
#pragma unroll
            for (int c = 0; c < kD / 16; ++c) reinterpret_cast<float4*>(sums)[(c * kN + n) * 32 + lane] = {o[c][n][0], o[c][n][1], o[c][n][2], o[c][n][3]};
        }
    };
    float* const early = a.partial + ((int64_t)blockIdx.x * kWarps + warp) * kPiece;
    bool kept = false, from_start = at.t == 0;
    if (lane < 2) s_piece[2 * warp + lane].tile0 = -1;
    __syncwarp();
    int to = 0, from = 0;                                                          // stages: of the next copy, of the next tile's work
    for (int i = 1 - kStages; i < 0 || at.place < span; ++i) {
        if (i >= 0) {
            copies_wait<kStages - 2>();
            __syncwarp();
        }
        if (in.place < span) {
            copy_tile(to);
            next_tile();
            to = to + 1 == kStages ? 0 : to + 1;
        }
        copies_end();
        if (i < 0) {
            if (i == -1 && at.place < span) begin_segment(true);
            continue;
        }
        work_on(from);
        from = from + 1 == kStages ? 0 : from + 1;
        const bool ends = at.t + 1 == at.tiles, last = at.place + 1 + (ends ? kBegin : 0) >= span;
        if (ends || last) {
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
                    if (kE4m3) {
                        const float back = power_of_2(-exponent(v_up[n][j]));
#pragma unroll
                        for (int c = 0; c < kD / 16; ++c) { o[c][n][j] *= back; o[c][n][2 + j] *= back; }
                    }
                }
            if (ends && from_start) {                                               // the whole segment was this warp's
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    const float2 inv = at.len > 0 ? float2{reciprocal(l[n][0]), reciprocal(l[n][1])} : float2{0.f, 0.f};
                    // A copy of the loop for bf16 and one for codes take less time than a branch in it (8 sequences of up to 4096 tokens 16.2 -> 15.5 us, 256 of
                    // up to 512 13.7 -> 13.3), except where two blocks of e4m3 tokens a turn leave no registers for it (131071 tokens 34.4 -> 35.8)
                    constexpr int kAtOnce = kE4m3 && kM == 2 ? 1 : kD / 16;
#pragma unroll
                    for (int c = 0; c < kD / 16; c += kAtOnce)
                        result.store<kE4m3, kAtOnce>(at.b, at.head * group + at.part * kHeads, min(kHeads, group - at.part * kHeads), c, n,
                                                     [&](int i) { return float4{o[c + i][n][0], o[c + i][n][1], o[c + i][n][2], o[c + i][n][3]}; }, inv);
                }
            } else {
                if (lane == 0)
                    s_piece[2 * warp + last] = {begin + at.place - at.t, at.tiles, at.b, at.head * group + at.part * kHeads, min(kHeads, group - at.part * kHeads)};
                if (last) kept = true;                                             // stays in registers until the rings are done with
                else keep_piece(false, early);
            }
        }
        ++at.place;
        if (++at.t == at.tiles) {
            at.t = 0;
            from_start = true;
            if (!next_segment(at) && !last) {
                at.len = within(after_len, most);
                at.tiles = tiles_of(at.len);
                if (at.b + 1 < a.batch) after_len = ld_dep(a.lens + at.b + 1);
            }
            if (!last) begin_segment(false);
        }
    }

    // ---- pieces of a segment in this CTA ------------------------------------------------------------------------------
    copies_wait<0>();
    __syncwarp();
    if (kept) keep_piece(true, reinterpret_cast<float*>(my_ring));
    __syncthreads();
    // A lane for a piece (two per warp, the second its last), every warp for itself: runs of pieces of one segment.
    const int64_t seg = lane < 2 * kWarps ? s_piece[lane].tile0 : -1, seg_end = seg + (lane < 2 * kWarps ? s_piece[lane].tiles : 0);
    const uint32_t there = __ballot_sync(0xffffffffu, seg >= 0), below = there & ((1u << lane) - 1);
    const int64_t prev = __shfl_sync(0xffffffffu, seg, below ? 31 - __clz(below) : lane);
    const bool first = seg >= 0 && (below == 0 || prev != seg);
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    // ... and the one that other CTAs began, the one that others go on with
    const uint32_t open0 = __ballot_sync(0xffffffffu, first && seg < cta0), open1 = __ballot_sync(0xffffffffu, first && seg >= cta0 && seg_end > cta1);
    constexpr int kUnits = kPiece / 4;                                             // fragments of a lane: two heads, two channels
    constexpr int kOut = kPiece + 2 * kHeads;
    float* const pieces = a.partial + (int64_t)gridDim.x * kWarps * kPiece;         // [CTA][2][sums | m | l]
    if (warp == 0 && seg >= 0) s_entry[__popc(below)] = lane;
    // the weights of a run's pieces, and their part of its sum of weights: a warp for a query head
    for (int col = warp; col < kHeads; col += kWarps) {
        const float pm = seg >= 0 ? s_m[lane][col] : kNone, pl = seg >= 0 ? s_l[lane][col] : 0.f;
        float top = kNone;
        for (uint32_t left = firsts; left; left &= left - 1) {
            const uint32_t rest = left & (left - 1), members = there & (0u - (left & (0u - left))) & (rest ? (rest & (0u - rest)) - 1 : 0xffffffffu);
            const bool in_run = members >> lane & 1;
            const float t = warp_max(in_run ? pm : kNone);
            if (in_run) top = t;
        }
        if (seg >= 0) {
            const float f = exp2_approx(pm - top);
            s_f[lane][col] = f;
            s_l[lane][col] = f * pl;
            s_m[lane][col] = top;
        }
    }
    __syncthreads();
    uint32_t left = firsts;
    int run = 0;
#pragma unroll 1
    for (int x = warp; x < __popc(firsts) * (kUnits / 32); x += kWarps) {          // a warp for the fragments of 16 channels and 8 heads
        for (; run < x / (kUnits / 32); ++run) left &= left - 1;
        const int at_first = __ffs(left) - 1, frag = x % (kUnits / 32), n = frag % kN, col = n * 8 + 2 * t4;
        const uint32_t rest = left & (left - 1), members = there & ~((1u << at_first) - 1) & (rest ? (rest & (0u - rest)) - 1 : 0xffffffffu);
        const int k0 = __popc(there & ((1u << at_first) - 1)), k1 = k0 + __popc(members);
        float2 sum = {0.f, 0.f};
        float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = k0; k < k1; ++k) {
            const int e = s_entry[k];
            const float2 f = *reinterpret_cast<const float2*>(&s_f[e][col]), pl = *reinterpret_cast<const float2*>(&s_l[e][col]);
            const float* from = (e & 1) ? reinterpret_cast<const float*>(ring + (e >> 1) * (kStages * S::kStageBytes))
                                        : a.partial + ((int64_t)blockIdx.x * kWarps + (e >> 1)) * kPiece;
            const float4 w = reinterpret_cast<const float4*>(from)[frag * 32 + lane];
            sum.x += pl.x; sum.y += pl.y;
            v.x += f.x * w.x; v.y += f.y * w.y; v.z += f.x * w.z; v.w += f.y * w.w;
        }
        const uint32_t bit = 1u << at_first;
        if ((open0 | open1) & bit) {
            float* out = pieces + ((int64_t)blockIdx.x * 2 + (open1 & bit ? 1 : 0)) * kOut;
            reinterpret_cast<float4*>(out)[frag * 32 + lane] = v;
            if (frag < kN && g == 0) {                                             // (the first channels' fragments have every head once)
                *reinterpret_cast<float2*>(out + kPiece + col) = *reinterpret_cast<const float2*>(&s_m[at_first][col]);
                *reinterpret_cast<float2*>(out + kPiece + kHeads + col) = sum;
            }
        } else {
            const Piece p = s_piece[at_first];
            result.store<kE4m3, 1>(p.b, p.head0, p.heads, frag / kN, n, [&](int) { return v; }, {reciprocal(sum.x), reciprocal(sum.y)});
        }
    }

    // ---- segments that other CTAs have pieces of: the last one to come joins them --------------------------------------
    // More than kJoin of them in two steps: first groups of about the square root of their number, each by the group's last CTA.  (One SM
    // reads some 40 GB/s of pieces: 74 of 8 KB took it 15 us.)
    if ((open0 | open1) == 0) return;
    auto group_of = [](int count) { return count <= kJoin ? count : (int)ceilf(sqrtf((float)count)); };
    __syncthreads();
    if (tid < 2) {
        bool last = false;
        if (tid == 0 ? open0 : open1) {
            const Piece p = s_piece[__ffs(tid == 0 ? open0 : open1) - 1];
            const int c0 = apart ? blockIdx.x - own_part : (int)quotient(p.tile0, share);
            const int count = apart ? own_parts : (int)quotient(p.tile0 + p.tiles - 1, share) - c0 + 1;
            const int size = group_of(count), first = size == count ? 0 : ((int)blockIdx.x - c0) / size * size, members = min(size, count - first);
            s_cta0[tid] = c0;
            s_first[tid] = first;
            s_ctas[tid] = count;
            int* const counter = a.counters + 2 * (c0 + first) + (first == 0);     // of the slot that the group's first piece is in
            last = arrive(counter) == members - 1;
            if (last) *counter = 0;                                                // for the next call
        }
        s_last[tid] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < 2; ++w) {
        if (!s_last[w]) continue;
        const Piece p = s_piece[__ffs(w == 0 ? open0 : open1) - 1];
        const int c0 = s_cta0[w], count = s_ctas[w], size = group_of(count);
        // the first CTA's piece is its second one, the others' their first
        float* const piece0 = pieces + ((int64_t)c0 * 2 + 1) * kOut;
        float* const piece1 = pieces + ((int64_t)c0 * 2) * kOut;
        auto piece_of = [&](int i) { return i == 0 ? piece0 : piece1 + (uint32_t)i * (2 * kOut); };
        // kSlices threads share a fragment's pieces
        constexpr int kSlices = S::kThreads > kUnits ? S::kThreads / kUnits : 1, kPerThread = kUnits > S::kThreads ? kUnits / S::kThreads : 1;
        const int slice = tid / kUnits;
        int start = s_first[w], stride = 1, n = min(size, count - start);
#pragma unroll 1
        for (;;) {
            uint4 raw[kJoin / kSlices];
            auto ask = [&](int unit) {
#pragma unroll
                for (int i = 0; i < kJoin / kSlices; ++i)
                    if (slice + i * kSlices < n) raw[i] = ld_dep_l2(reinterpret_cast<const uint4*>(piece_of(start + (slice + i * kSlices) * stride)) + unit);
            };
            for (int col = warp; col < kHeads; col += kWarps) {                    // a warp for a query head, a lane for a piece
                float pm = kNone, pl = 0.f;
                if (lane < n) {
                    pm = ld_dep_l2(piece_of(start + lane * stride) + kPiece + col);
                    pl = ld_dep_l2(piece_of(start + lane * stride) + kPiece + kHeads + col);
                }
                const float top = warp_max(pm), f = exp2_approx(pm - top);
                float sum = f * pl;
                for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (lane < n) s_share[lane][col] = f;
                if (lane == 0) { s_top[col] = top; s_sum[col] = sum; }
            }
            __syncthreads();
            float4 v[kPerThread];
#pragma unroll
            for (int k = 0; k < kPerThread; ++k) {
                const int unit = (tid + k * S::kThreads) % kUnits, col = (unit >> 5) % kN * 8 + 2 * t4;
                v[k] = {0.f, 0.f, 0.f, 0.f};
                ask(unit);
#pragma unroll
                for (int i = 0; i < kJoin / kSlices; ++i)
                    if (slice + i * kSlices < n) {
                        const float2 f = *reinterpret_cast<const float2*>(&s_share[slice + i * kSlices][col]);
                        v[k].x += f.x * __uint_as_float(raw[i].x); v[k].y += f.y * __uint_as_float(raw[i].y);
                        v[k].z += f.x * __uint_as_float(raw[i].z); v[k].w += f.y * __uint_as_float(raw[i].w);
                    }
            }
            if (kSlices > 1) {
                float4* const sums = reinterpret_cast<float4*>(ring);
                if (slice > 0) sums[tid - kUnits] = v[0];
                __syncthreads();
                if (slice == 0) {
#pragma unroll
                    for (int k = 1; k < kSlices; ++k) {
                        const float4 y = sums[(k - 1) * kUnits + tid];
                        v[0].x += y.x; v[0].y += y.y; v[0].z += y.z; v[0].w += y.w;
                    }
                }
            }
            const bool all = size == count || stride > 1;
            if (slice == 0) {
#pragma unroll
                for (int k = 0; k < kPerThread; ++k) {
                    const int unit = tid + k * S::kThreads, frag = unit >> 5, n8 = frag % kN, col = n8 * 8 + 2 * t4;
                    const float2 top = *reinterpret_cast<const float2*>(&s_top[col]), sum = *reinterpret_cast<const float2*>(&s_sum[col]);
                    if (all) {
                        result.store<kE4m3, 1>(p.b, p.head0, p.heads, frag / kN, n8, [&](int) { return v[k]; }, {reciprocal(sum.x), reciprocal(sum.y)});
                    } else {                                                       // in place of the group's first
                        float* const out = piece_of(start);
                        reinterpret_cast<float4*>(out)[unit] = v[k];
                        if (frag < kN && g == 0) {
                            *reinterpret_cast<float2*>(out + kPiece + col) = top;
                            *reinterpret_cast<float2*>(out + kPiece + kHeads + col) = sum;
                        }
                    }
                }
            }
            __syncthreads();                                                       // s_share and its companions are free again
            if (all) break;
            if (tid == 0) {
                int* const counter = a.counters + 2 * kMaxCtas + c0;
                s_again = arrive(counter) == (count + size - 1) / size - 1;
                if (s_again) *counter = 0;
            }
            __syncthreads();
            if (!s_again) break;
            start = 0;
            stride = size;
            n = (count + size - 1) / size;
        }
    }
}

int attention_ctas() { return sm_count() < kMaxCtas ? sm_count() : kMaxCtas; }

template <class S>
cudaError_t launch(const AttnArgs& a, int group, int parts, cudaStream_t stream) {
    auto kern = paged_attention_kernel<S>;
    static std::atomic<uint64_t> ready{0};              // devices whose copy of the kernel may take this much shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kRing);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)attention_ctas());
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kRing;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.numAttrs = pdl_attribute(attr);
    cfg.attrs = attr;
    return counted(cudaLaunchKernelEx(&cfg, kern, a, group, parts));
}

// Calls f with the kernel's shape for these heads: channels rounded up to 64, 128 or 256; 16 query heads at a time for groups of
// more than 8 (256 channels: 8, whose sums fill the registers), the rest of a larger group as segments of their own.
template <class F>
auto with_shape(bool e4m3, int64_t dim, int64_t group, F&& f) {
    // (16 at a time take a warp 1.5 us for 16 tokens of an e4m3 cache, 8 at a time 1.6 us for 32; so an odd number of eights goes one by one)
    const bool wide = group > 8 && (!e4m3 || (group + 7) / 8 % 2 == 0);
    if (e4m3) {
        if (dim <= 64) return wide ? f(Shape<true, 64, 2, 1, 8, 6>()) : f(Shape<true, 64, 1, 2, 16, 3>());
        if (dim <= 128) return wide ? f(Shape<true, 128, 2, 1, 8, 6>()) : f(Shape<true, 128, 1, 2, 8, 3>());
        return f(Shape<true, 256, 1, 1, 8, 3>());
    }
    if (dim <= 64) return wide ? f(Shape<false, 64, 2, 1, 8, 6>()) : f(Shape<false, 64, 1, 2, 8, 3>());
    if (dim <= 128) return wide ? f(Shape<false, 128, 2, 1, 8, 3>()) : f(Shape<false, 128, 1, 1, 8, 3>());
    return f(Shape<false, 256, 1, 1, 4, 3>());
}

}  // namespace

size_t paged_attention_scratch(int64_t heads, int64_t kv_heads, int64_t dim, bool e4m3) {
    return with_shape(e4m3, dim, heads / kv_heads, [](auto s) { return scratch_floats<decltype(s)>(attention_ctas()) * sizeof(float); });
}

cudaError_t launch_paged_attention(const AttnArgs& a, cudaStream_t stream) {
    const int group = a.heads / a.c.kv_heads;
    return with_shape(a.c.e4m3, a.c.dim, group, [&](auto s) {
        using S = decltype(s);
        const int parts = (group + S::kHeads - 1) / S::kHeads;
        AttnArgs x = a;
        x.by_page = Divisor(a.c.block_size);
        x.by_segments = Divisor(a.c.kv_heads * parts);
        x.by_parts = Divisor(parts);
        return launch<S>(x, group, parts, stream);
    });
}

}  // namespace fp8lin
