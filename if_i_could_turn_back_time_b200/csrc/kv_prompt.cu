// Attention over the 8-bit cache, many query rows per key head (prompts and parts of prompts): tcgen05.
//
// A CTA has 256 rows (query, head of the group) of a key head as two tiles of 128 and walks along the keys in tiles of 64.
// Four warps turn a tile's codes into fp16 operands in shared memory, once for both row tiles; a warp for each row tile issues
// S = Q K^T and O += P V (M = 128, N = 64 and N = D, accumulators in tensor memory); sixteen warps, two threads per row,
// turn scores into weights, which go back to tensor memory as the A operand of the second product; one plans.  Block scales
// never touch the operands: a key block's scale multiplies its columns of S in fp32, a value block's goes into the exponent,
//   t = s ks scale log2(e) + log2(vs),  p = 2^(t - ref),  O = sum p v_code,  l = sum p / vs,  out = O / l,
// and O is only rescaled when a row's largest t has grown by more than 2^8 since its reference was set (kLift, kGrowth).
//
// 1024 tokens behind 15360 cached ones, 64 query and 8 key heads of 128: 540 us in a short burst, 573 once the power cap holds the clock
// at 1.84 GHz (990 and 930 TFLOP/s); a prompt of 2048 tokens, 32 heads: 79 us.
// A step of 64 keys takes about 2100 clocks, of which the tensor core needs 1150 and the exponentials' unit 1024; the rest is the
// latency of a row's chain scores -> maxima -> weights -> tensor memory (one thread per row: 664 us; four warps a tile).  At 80 registers a
// thread all instances spill a little: 36 bytes stored, 48 loaded.
#include "kv_attend.cuh"

namespace jqkv {

using namespace jqta;

namespace prompt {

constexpr int kThreads = 768;      // warps 0-15: weights, 16-19: codes to operands, 20 and 21: matrix instructions, 22: segments
constexpr int kRows = kPromptRows, kKeys = 64;
constexpr int kStages = 4;         // of the rings of key and value operands
constexpr int kSegments = 32;      // planned at once
constexpr int kPairCost = 6;       // what a pair costs besides its key tiles, in units of one: queries, outputs, hand-over
// A row's reference is set 2^7 below its largest weight, and O rescaled when that has grown by more than 2^8: weights are fp16 numbers up to
// 2^15, with eleven bits down to 2^-21 of the largest at least.  (The sum of 16384 weights of e^-11 to e^-17 behind a strong token whose value
// is small: off by 0.1 % at most with fp16 outputs, with the reference at the largest by 0.2 to 2.5 %.  us of the two cases above with 2^7 and 2^8:
// 573 and 80; 2^10 and 2^5: 578 and 82; 2^14 and 2: 587 and 83; 0 and 2^8: 568 and 80.)
constexpr float kLift = 7.f, kGrowth = 8.f;
constexpr int kScaleSlots = 8;     // tiles whose scales are kept: at most five are in use (four operands ahead of the scores)
constexpr int kQTmem = 64;         // values of a query row in tensor memory; the others, at D = 128, lie in shared memory

template <int D>
struct Shape {
    static constexpr int kLbo = kKeys * 16 + 32;             // bytes between 16-byte slices of the keys: 32 more than they take,
    static constexpr int kKBytes = D / 8 * kLbo;             //   so that the eight lanes of a store phase meet different banks
    static constexpr int vLbo = D * 16 + 64;                 // the same between slices of 8 keys of the values
    static constexpr int vBytes = kKeys / 8 * vLbo;
    static constexpr int qBytes = D > kQTmem ? (D - kQTmem) * 2 * 128 : 0;     // per row tile
    static constexpr int smem = kStages * (kKBytes + vBytes) + 2 * qBytes;
    static constexpr int part = kRows * D + 2 * kRows;       // floats of a part
};
// Tensor memory of a row tile: the output's D columns at 0, scores, weights and queries behind them
constexpr int kColS = 128, kColP = 192, kColQ = 224, kColTile = 256;

__device__ __forceinline__ void mma_f16_ss(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0;\n"
                 "  @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}

__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return r;
}
// Two fp32 values in a register pair
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair2(uint32_t a, uint32_t b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float2 unpair2(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Keys that the rows of a tile see, rounded down to a unit at their beginning.
struct Range {
    int see, lo, hi, units;        // see: lo before it was rounded; units: kPairCost and the key tiles
};
__device__ __forceinline__ Range range_of(const AttendArgs &p, int len, int n, int tile) {
    const int first = len - n;
    const int q0 = (int)((uint32_t)tile * kRows / (uint32_t)p.G), q1 = min(n - 1, (int)(((uint32_t)(tile + 1) * kRows - 1) / (uint32_t)p.G));
    Range r;
    r.hi = max(0, min(len, first + q1 + 1));
    r.see = first_seen(p, first + q0);
    r.lo = min(r.see, r.hi) & ~(kKeys - 1);
    r.units = kPairCost + max(1, (r.hi - r.lo + kKeys - 1) / kKeys);
    return r;
}
// (n * G is at most 2^30 where max_new is what it says; a longer sequence has its first 2^30 rows)
__device__ __forceinline__ int tiles_of(const AttendArgs &p, int n) { return (int)((min((long long)n * p.G, 1LL << 30) + kRows - 1) / kRows); }

// The segments of a CTA: units in the order (sequence, row tile, key head, unit), cut evenly.
struct Walk {
    long long cur, end, at;        // at: first unit of (seq, tile)
    int seq, tile, n, len, row0, tiles;
    Range range;
    int head, u0, u1;              // of the segment: key head, key tiles
    __device__ __forceinline__ void sequence(const AttendArgs &p) {
        n = p.b.count(seq, row0);
        len = p.b.length(seq);
        tiles = tiles_of(p, n);
    }
    __device__ __forceinline__ bool next(const AttendArgs &p) {
        while (cur < end) {
            while (tiles == 0 || cur >= at + (long long)range.units * p.H) {
                if (tiles) at += (long long)range.units * p.H;
                if (++tile >= tiles) {
                    ++seq;
                    tile = 0;
                    sequence(p);
                }
                if (tiles) range = range_of(p, len, n, tile);
            }
            const long long in = cur - at;
            head = (int)quotient(in, range.units);
            u0 = (int)(in - (long long)head * range.units);
            u1 = (int)min((long long)range.units, u0 + (end - cur));
            cur += u1 - u0;
            // from here on in key tiles: the first units of a pair stand for none
            u0 = max(0, u0 - kPairCost);
            u1 -= kPairCost;
            if (u1 > u0) return true;
        }
        return false;
    }
};

// A segment, as the planning warp hands it to the others.
struct Segment {
    int tiles, key0, see, hi;      // key tiles, first key, begin and end of the keys that its rows see
    int seq, head, row0, n, len;   // row0, n: the sequence's rows of the call's tensors
    int flat0, rows;               // first of the rows (query, head of the group) among the sequence's, and how many
    int all, w0, w1, slot;         // the whole of a pair, or a part: CTAs that have one, and the place of this one's
};

template <int D, bool E4M3>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ AttendArgs p) {
    using S = Shape<D>;
    constexpr int H = D / 2;                                 // values of a row that a thread loads, scales and stores
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[4 * kStages + 2 * 5];
    __shared__ __align__(16) float s_scales[kScaleSlots][4][4];    // [.][group]: scale of the keys (negative: not there), log2(vs), 1 / vs
    __shared__ float s_top[2][2][kRows];                     // [parity][half][row]
    __shared__ Segment s_seg[kSegments];
    __shared__ long long s_sum[8], s_at;
    __shared__ int s_err, s_seq, s_tile, s_last, s_count;
    __shared__ uint32_t s_tmem;

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t b0 = smem_u32(bars);
    auto kfull = [&](int s) { return b0 + 8 * s; };
    auto kfree = [&](int s) { return b0 + 8 * (kStages + s); };
    auto vfull = [&](int s) { return b0 + 8 * (2 * kStages + s); };
    auto vfree = [&](int s) { return b0 + 8 * (3 * kStages + s); };
    auto qfull = [&](int w) { return b0 + 8 * (4 * kStages + w); };
    auto sfull = [&](int w) { return b0 + 8 * (4 * kStages + 2 + w); };
    auto sfree = [&](int w) { return b0 + 8 * (4 * kStages + 4 + w); };
    auto pfull = [&](int w) { return b0 + 8 * (4 * kStages + 6 + w); };
    auto odone = [&](int w) { return b0 + 8 * (4 * kStages + 8 + w); };

    // ---- this CTA's units: a group of threads for each sequence, tiles in turn over its threads
    const int spread = p.b.S >= 256 ? 1 : 256 / p.b.S, per = (p.b.S + 255) / 256;
    int my_seq = 0, my_seqs = 0, my_tile = 0, my_tiles = 0;
    long long mine = 0;
    auto tiles_sum = [&](int i, int t0, int t1) {
        int row0;
        const int n = p.b.count(i, row0), len = p.b.length(i), tiles = tiles_of(p, n);
        long long sum = 0;
        for (int t = t0; t < min(t1, tiles); ++t) sum += (long long)range_of(p, len, n, t).units * p.H;
        return sum;
    };
    if (tid < 256) {
        if (spread == 1) {
            my_seq = min(p.b.S, tid * per);
            my_seqs = min(p.b.S, my_seq + per) - my_seq;
            my_tiles = 0x7fffffff;
        } else {
            my_seq = tid / spread;
            my_seqs = my_seq < p.b.S ? 1 : 0;
            if (my_seqs) {
                int row0;
                const int tiles = tiles_of(p, p.b.count(my_seq, row0)), c = (tiles + spread - 1) / spread;
                my_tile = tid % spread * c;
                my_tiles = my_tile + c;
            }
        }
        for (int i = 0; i < my_seqs; ++i) mine += tiles_sum(my_seq + i, my_tile, my_tiles);
    }
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31 && warp < 8) s_sum[warp] = before;
    if (tid == 0) {
        s_err = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(kfull(s), 4);
            mbar_init(vfull(s), 4);
            mbar_init(kfree(s), 2);
            mbar_init(vfree(s), 2);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(qfull(w), 8);
            mbar_init(sfull(w), 1);
            mbar_init(sfree(w), 8);
            mbar_init(pfull(w), 8);
            mbar_init(odone(w), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < 8; ++w) {
        if (w == warp) before += total - mine;
        total += s_sum[w];
    }
    if (total == 0) return;
    const long long fit = quotient(total + p.least - 1, p.least);
    const int W = fit < (long long)gridDim.x ? (int)fit : (int)gridDim.x;
    if ((int)blockIdx.x >= W) return;
    const Shares shares(total, W);
    const long long cur = shares.first(blockIdx.x);
    if (tid < 256 && cur >= before && cur < before + mine) {
        long long at = before;
        for (int i = 0; i < my_seqs; ++i) {
            int row0;
            const int n = p.b.count(my_seq + i, row0), len = p.b.length(my_seq + i), tiles = tiles_of(p, n);
            for (int t = my_tile; t < min(my_tiles, tiles); ++t) {
                const long long u = (long long)range_of(p, len, n, t).units * p.H;
                if (cur >= at && cur < at + u) {
                    s_seq = my_seq + i;
                    s_tile = t;
                    s_at = at;
                }
                at += u;
            }
        }
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int *err = &s_err;
    auto wait = [&](uint32_t bar, uint32_t parity) {          // (converged again behind it: what follows is often the whole warp's)
        mbar_wait(bar, parity, err);
        __syncwarp();
    };
    unsigned char *const kring = smem, *const vring = smem + kStages * S::kKBytes, *const qmem = vring + kStages * S::vBytes;

    // The next segment, in batches that the planning warp fills.  How often a warp gets to a barrier goes by the segments alone, so that
    // the barriers are met even after a wait that gave up.
    int seg = kSegments, segs = kSegments;
    auto batch_sync = [&]() { asm volatile("bar.sync 10, 736;" ::: "memory"); };
    auto next_segment = [&]() -> const Segment * {
        if (seg == segs) {
            if (segs < kSegments) return nullptr;          // (the last batch is not full)
            batch_sync();                                  // every warp is done with the batch before
            batch_sync();                                  // the next one is there
            segs = s_count;
            seg = 0;
            if (segs == 0) return nullptr;
        }
        return &s_seg[seg++];
    };
    // Registers: 768 x 80 at launch = 512 x 80 + 128 x 96 + 128 x 64
    if (warp < 16) {
        // ============ scores to weights: two threads per row, each with 32 of a tile's 64 keys and half of the row's values ============
        const int w = warp >> 3, half = warp >> 2 & 1, r = (warp & 3) * 32 + lane, row = w * 128 + r;
        const int pair_bar = 1 + w * 4 + (warp & 3);                                     // the two warps that have the same rows
        const uint32_t mine_t = tmem + w * kColTile + ((uint32_t)(warp & 3) << 21);      // their 32 lanes of tensor memory
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory"); };
        uint32_t it = 0;                                   // tiles of this row tile so far
        int slot = 0;                                      // of the scales
        while (const Segment *sg = next_segment()) {
            const int tiles = sg->tiles, rows = sg->rows;
            const bool active = w == 0 || rows > 128;
            const bool there = row < rows;
            const int fr = sg->flat0 + (there ? row : 0), j = fr / p.G, hq = sg->head * p.G + fr % p.G;
            float ref = -INFINITY, l = 0.f, qs = 0.f;
            if (active) {
                // half of the query row, divided by a power of two that brings the row into fp16's range
                // (a row that is not there reads the tile's first; nothing comes of it)
                const unsigned short *at = reinterpret_cast<const unsigned short *>(p.q) + (sg->row0 + j) * p.st + hq * p.sh + half * H;
                uint4 raw[H / 8];
                if ((p.st | p.sh) % 8 == 0 && (reinterpret_cast<uintptr_t>(p.q) & 15u) == 0) {
#pragma unroll
                    for (int c = 0; c < H / 8; ++c) raw[c] = __ldg(reinterpret_cast<const uint4 *>(at) + c);
                } else {
#pragma unroll
                    for (int c = 0; c < H / 8; ++c) {
                        uint32_t x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = at[c * 8 + 2 * k] | (uint32_t)at[c * 8 + 2 * k + 1] << 16;
                        raw[c] = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                auto value = [&](uint32_t x, int hi_half) -> float {
                    const unsigned short u = (unsigned short)(hi_half ? x >> 16 : x & 0xffffu);
                    return p.dtype == JQ_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float((uint32_t)u << 16);
                };
                float amax = 0.f;
#pragma unroll
                for (int c = 0; c < H / 8; ++c) {
                    const uint32_t x[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(fabsf(value(x[k], 0)), fabsf(value(x[k], 1))));
                }
                s_top[1][half][row] = amax;
                pair_sync();
                amax = fmaxf(amax, s_top[1][half ^ 1][row]);
                pair_sync();
                const int e = query_exponent(amax);
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                qs = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale;
#pragma unroll
                for (int c4 = 0; c4 < H / 32; ++c4) {
                    uint32_t h[16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint4 u = raw[c4 * 4 + c];
                        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) h[c * 4 + k] = pack_h2(value(x[k], 0) * down, value(x[k], 1) * down);
                    }
                    if (D <= kQTmem || half == 0) {
                        tmem_st16(mine_t + kColQ + half * (H / 2) + c4 * 16, h);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint4 *>(qmem + w * S::qBytes + (c4 * 4 + c) * 2048 + r * 16) =
                                make_uint4(h[c * 4], h[c * 4 + 1], h[c * 4 + 2], h[c * 4 + 3]);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull(w));
            }
            // columns of the thread that its row sees, counted from its first
            int last = (there ? sg->len - sg->n + j : -1) - sg->key0 - half * 32;
            bool ready = false;                            // the next scores are there
            for (int i = 0; i < tiles; ++i, last -= kKeys) {
                if (active) {
                    if (!__all_sync(0xffffffffu, ready)) wait(sfull(w), it & 1);
                    tc_fence_after();
                    uint32_t s[32];
                    tmem_ld32(mine_t + kColS + half * 32, s);
                    const float4 sc0 = *reinterpret_cast<const float4 *>(s_scales[slot][half * 2]),
                                 sc1 = *reinterpret_cast<const float4 *>(s_scales[slot][half * 2 + 1]);
                    const int first = p.window > 0 ? last - p.window + 1 : 0;
                    const bool edge = last < 31 || first > 0 || sc0.x < 0.f || sc1.x < 0.f;
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sfree(w));
                    if (__any_sync(0xffffffffu, edge)) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (c > last || c < first || (c < 16 ? sc0.x : sc1.x) < 0.f) s[c] = 0xff800000u;
                    }
                    float m0 = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])), m1 = fmaxf(__uint_as_float(s[16]), __uint_as_float(s[17]));
#pragma unroll
                    for (int c = 2; c < 16; c += 2) {
                        m0 = max3(m0, s[c], s[c + 1]);
                        m1 = max3(m1, s[16 + c], s[17 + c]);
                    }
                    // (never 0, which keys of zeros and tiny queries give: a masked score of -infinity times it would be NaN)
                    const float f0 = fmaxf(fabsf(sc0.x) * qs, 1.17549435e-38f), f1 = fmaxf(fabsf(sc1.x) * qs, 1.17549435e-38f);
                    float top = fmaxf(fmaf(m0, f0, sc0.y), fmaf(m1, f1, sc1.y));
                    float(*const tops)[kRows] = s_top[it & 1];
                    tops[half][row] = top;
                    pair_sync();
                    top = fmaxf(top, tops[half ^ 1][row]);           // (NaN is neither's maximum, and comes back in the sums)
                    if (i == 0) {
                        ref = fmaxf(top - kLift, -INFINITY);
                    } else if (__any_sync(0xffffffffu, top > ref + (kLift + kGrowth))) {
                        const float to = top > ref + (kLift + kGrowth) ? top - kLift : ref;
                        const float a = to == -INFINITY ? 1.f : ex2(ref - to);
                        ref = to;
                        l *= a;
                        wait(odone(w), (it & 1) ^ 1);
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < H / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(mine_t + half * H + c * 16, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * a);
                            tmem_st16(mine_t + half * H + c * 16, o);
                        }
                        tmem_wait_st();
                    }
                    const float base = ref == -INFINITY ? 0.f : -ref;
                    float g0 = f0, g1 = f1, add0 = sc0.y + base, add1 = sc1.y + base;
                    if (fabsf(base) > 8192.f) {
                        // exponents so large that the rounding of log2(vs) - ref would show in the weights: formed as the maximum was,
                        // then the difference
#pragma unroll
                        for (int c = 0; c < 32; ++c) s[c] = __float_as_uint(fmaf(__uint_as_float(s[c]), c < 16 ? f0 : f1, c < 16 ? sc0.y : sc1.y));
                        g0 = g1 = 1.f;
                        add0 = add1 = base;
                    }
                    __syncwarp();
                    // (asked here, needed behind the exponentials: whether the weights of the tile before have been used)
                    const bool used = mbar_test(odone(w), (it & 1) ^ 1);
                    uint32_t h[16];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const uint64_t f2 = n ? pair2(g1, g1) : pair2(g0, g0), a2 = n ? pair2(add1, add1) : pair2(add0, add0);
                        uint64_t sum = 0;
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            const float2 e = unpair2(fma2(pair2(s[16 * n + c], s[16 * n + c + 1]), f2, a2));
                            const float x = ex2(e.x), y = ex2(e.y);
                            sum = add2(sum, pair2(x, y));
                            h[8 * n + c / 2] = pack_h2(x, y);
                        }
                        const float2 sums = unpair2(sum);
                        l = fmaf(sums.x + sums.y, n ? sc1.z : sc0.z, l);
                    }
                    if (!__all_sync(0xffffffffu, used)) wait(odone(w), (it & 1) ^ 1);
                    tc_fence_after();
                    tmem_st16(mine_t + kColP + half * 16, h);
                    ready = mbar_test(sfull(w), (it & 1) ^ 1);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pfull(w));
                    ++it;
                }
                if (++slot == kScaleSlots) slot = 0;
            }
            // ---- outputs, or a part of them
            const bool all = sg->all != 0;
            float *part = p.parts + (size_t)sg->slot * S::part;
            if (active) {
                pair_sync();
                s_top[0][half][row] = l;
                pair_sync();
                l += s_top[0][half ^ 1][row];
                pair_sync();
                const size_t out_at = ((size_t)(sg->row0 + j) * p.H * p.G + hq) * D + half * H;
                if (there && half == 0) {
                    if (!all) {
                        part[kRows * D + row] = ref;
                        part[kRows * D + kRows + row] = l;
                    } else if (p.lse) {
                        p.lse[out_at / D] = lse_of(ref, l);
                    }
                }
                const float inv = inverse(l);
                wait(odone(w), (it & 1) ^ 1);
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < H / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16(mine_t + half * H + c * 16, o);
                    tmem_wait_ld();
                    if (there) {
#pragma unroll
                        for (int k = 0; k < 16; k += 8) {
                            float v[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) v[x] = __uint_as_float(o[k + x]);
                            if (all) {
                                store8(p, out_at + c * 16 + k, v, inv);
                            } else {                       // [four values][row]: a warp's rows are adjacent
                                float4 *dst = reinterpret_cast<float4 *>(part) + (half * H + c * 16 + k) / 4 * kRows + row;
                                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                                dst[kRows] = make_float4(v[4], v[5], v[6], v[7]);
                            }
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();
            }
            if (!all) {
                // the last of the pair's CTAs to get here adds the parts, in their order
                const int w0 = sg->w0, w1 = sg->w1;
                __threadfence();
                asm volatile("bar.sync 9, 512;" ::: "memory");
                if (tid == 0) {
                    const int n = atomicAdd(p.counters + w0, 1);
                    s_last = n == w1 - w0;
                    if (s_last) p.counters[w0] = 0;
                }
                asm volatile("bar.sync 9, 512;" ::: "memory");
                if (s_last) {
                    __threadfence();
                    if (there) {
                        auto of = [&](int x) { return p.parts + (size_t)(2 * x + (x == w0 ? 1 : 0)) * S::part; };
                        float m = -INFINITY, lsum = 0.f;
                        for (int x = w0; x <= w1; ++x) m = fmaxf(m, __ldcg(of(x) + kRows * D + row));
                        const float base = m == -INFINITY ? 0.f : m;
                        for (int x = w0; x <= w1; ++x)
                            lsum = fmaf(__ldcg(of(x) + kRows * D + kRows + row), ex2(__ldcg(of(x) + kRows * D + row) - base), lsum);
                        const float f = inverse(lsum);
                        const size_t o = ((size_t)(sg->row0 + j) * p.H * p.G + hq) * D + half * H;
                        if (half == 0 && p.lse) p.lse[o / D] = lse_of(m, lsum);
#pragma unroll 1
                        for (int c = 0; c < H; c += 16) {
                            float v[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) v[k] = 0.f;
                            for (int x = w0; x <= w1; ++x) {
                                const float4 *y = reinterpret_cast<const float4 *>(of(x)) + (half * H + c) / 4 * kRows + row;
                                const float a = ex2(__ldcg(of(x) + kRows * D + row) - base);
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const float4 u = __ldcg(y + k * kRows);
                                    v[4 * k] = fmaf(u.x, a, v[4 * k]); v[4 * k + 1] = fmaf(u.y, a, v[4 * k + 1]);
                                    v[4 * k + 2] = fmaf(u.z, a, v[4 * k + 2]); v[4 * k + 3] = fmaf(u.w, a, v[4 * k + 3]);
                                }
                            }
#pragma unroll
                            for (int k = 0; k < 16; k += 8) store8(p, o + c + k, *reinterpret_cast<const float(*)[8]>(v + k), f);
                        }
                    }
                }
                asm volatile("bar.sync 9, 512;" ::: "memory");           // (s_last is read before the next segment writes it)
            }
        }
    } else if (warp < 20) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        // =============================== codes to operands: a warp per 16 keys of a tile ===============================
        const int cw = warp - 16, g = lane >> 2, t = lane & 3;
        constexpr int C = D / 32;
        int st = 0, slot = 0;
        uint32_t par = 1;                                  // (the first round finds every stage free)
        const uint32_t none = E4M3 ? 0u : 0x80808080u;     // code of 0
        while (const Segment *sg = next_segment()) {
            const int tiles = sg->tiles, key0 = sg->key0 + 16 * cw, see = sg->see, hi = sg->hi, head = sg->head, len = sg->len, seq = sg->seq;
            int id = -1;
            float kc = -1.f, vl = 0.f, vi = 1.f;
            auto look_up = [&](int first) {                // lane l: block and scales of tile first + l
                const int k = key0 + (first + lane) * kKeys;
                id = -1;
                // (16 keys that nobody sees are not looked at: their block may be another sequence's by now)
                if (first + lane < tiles && k < hi && k + 16 > see) id = p.b.block(seq, k);
                kc = -1.f;
                vl = 0.f;
                vi = 1.f;
                if (id >= 0) {
                    const size_t at = (size_t)id * p.H + head;
                    const float v = p.vs[at];
                    kc = p.ks[at];
                    vl = log2f(v);
                    vi = __fdividef(1.f, v);
                }
            };
            uint4 kr[C], vr[C];
            auto load = [&](const uint8_t *codes, int tile, uint4 (&x)[C]) {     // (ids of the 32 tiles that `tile` is one of)
                const int b = __shfl_sync(0xffffffffu, id, tile & 31);
                const int k = key0 + tile * kKeys;
                const uint4 *at = reinterpret_cast<const uint4 *>(codes + (((size_t)max(b, 0) * p.H + head) * p.b.T + (k & (p.b.T - 1))) * D) + lane;
#pragma unroll
                for (int c = 0; c < C; ++c) x[c] = b >= 0 ? __ldg(at + c * 32) : make_uint4(none, none, none, none);
            };
            look_up(0);
            load(p.keys, 0, kr);
            load(p.values, 0, vr);
            for (int i = 0; i < tiles; ++i) {
                const float kc_i = __shfl_sync(0xffffffffu, kc, i & 31), vl_i = __shfl_sync(0xffffffffu, vl, i & 31),
                            vi_i = __shfl_sync(0xffffffffu, vi, i & 31);
                if (i + 1 < tiles && ((i + 1) & 31) == 0) look_up(i + 1);
                wait(kfree(st), par);
                unsigned char *kd = kring + st * S::kKBytes + t * S::kLbo + (16 * cw + 4 * (g >> 1) + (g & 1)) * 16;
                // (in shared memory before the operand is announced: who waits for the scores made of it finds them there)
                if (lane == 0) *reinterpret_cast<float4 *>(s_scales[slot][cw]) = make_float4(kc_i, vl_i, vi_i, 0.f);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    uint4 a, b;
                    codes_to_h4<E4M3>(kr[c].x, a.x, a.y);
                    codes_to_h4<E4M3>(kr[c].y, a.z, a.w);
                    codes_to_h4<E4M3>(kr[c].z, b.x, b.y);
                    codes_to_h4<E4M3>(kr[c].w, b.z, b.w);
                    *reinterpret_cast<uint4 *>(kd + c * 4 * S::kLbo) = a;
                    *reinterpret_cast<uint4 *>(kd + c * 4 * S::kLbo + 32) = b;
                }
                if (i + 1 < tiles) load(p.keys, i + 1, kr);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(kfull(st));
                wait(vfree(st), par);
                unsigned char *vd = vring + st * S::vBytes + (2 * cw + (t >> 1)) * S::vLbo + g * 16 + (t & 1) * 8;
                uint32_t keep = 0xffffffffu;               // e4m3 has a NaN, and places behind the sequence's end may hold anything
                if (E4M3) {
                    const int left = len - (key0 + i * kKeys + 4 * t);
                    keep = left >= 4 ? 0xffffffffu : (left <= 0 ? 0u : (1u << 8 * left) - 1u);
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint32_t word[4] = {vr[c].x, vr[c].y, vr[c].z, vr[c].w};
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt) {
                        uint2 a;
                        codes_to_h4<E4M3>(E4M3 ? word[dt] & keep : word[dt], a.x, a.y);
                        *reinterpret_cast<uint2 *>(vd + (c * 32 + dt * 8) * 16) = a;
                    }
                }
                if (i + 1 < tiles) load(p.values, i + 1, vr);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(vfull(st));
                if (++st == kStages) { st = 0; par ^= 1; }
                if (++slot == kScaleSlots) slot = 0;
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp < 22) {
            // =============================== matrix instructions: a warp for each row tile ===============================
            // (One warp for both took 1080 clocks for a tile of each, waits and issue one after another, where the tensor core
            // needs 580.  The warp runs converged, see mma_f16_ts.)
            const int w = warp - 20;
            const uint32_t elected = elect_one();
            const uint32_t t0 = tmem + w * kColTile;
            const uint64_t kdesc = smem_desc(smem_u32(kring), S::kLbo, 128), vdesc = smem_desc(smem_u32(vring), S::vLbo, 128),
                           qdesc = smem_desc(smem_u32(qmem + w * S::qBytes), 2048, 128);
            constexpr uint32_t idesc_s = idesc_f16(128, kKeys), idesc_o = idesc_f16(128, D);
            int ks = 0, vs = 0;
            uint32_t kpar = 0, vpar = 0, qpar = 0, spar = 1, opar = 0;
            auto next_k = [&]() { if (++ks == kStages) { ks = 0; kpar ^= 1; } };
            auto next_v = [&]() { if (++vs == kStages) { vs = 0; vpar ^= 1; } };
            auto scores = [&]() {
                wait(kfull(ks), kpar);
                wait(sfree(w), spar);
                spar ^= 1;
                tc_fence_after();
                const uint64_t b = kdesc + (uint64_t)(ks * (S::kKBytes >> 4));
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    if (k < kQTmem / 16) mma_f16_ts(elected, t0 + kColS, t0 + kColQ + 8 * k, b + (uint64_t)(k * (2 * S::kLbo >> 4)), idesc_s, k > 0);
                    else mma_f16_ss(elected, t0 + kColS, qdesc + (uint64_t)((k - kQTmem / 16) * (4096 >> 4)),
                                    b + (uint64_t)(k * (2 * S::kLbo >> 4)), idesc_s, 1);
                }
                mma_commit(elected, sfull(w));
                mma_commit(elected, kfree(ks));
                next_k();
            };
            while (const Segment *sg = next_segment()) {
                const int tiles = sg->tiles, rows = sg->rows;
                if (w == 1 && rows <= 128) {       // the operands are the other tile's alone
                    for (int i = 0; i < tiles; ++i) {
                        wait(kfull(ks), kpar);
                        if (lane == 0) mbar_arrive(kfree(ks));
                        next_k();
                        wait(vfull(vs), vpar);
                        if (lane == 0) mbar_arrive(vfree(vs));
                        next_v();
                    }
                    continue;
                }
                wait(qfull(w), qpar);
                qpar ^= 1;
                scores();
                for (int i = 0; i < tiles; ++i) {
                    if (i + 1 < tiles) scores();
                    wait(vfull(vs), vpar);
                    wait(pfull(w), opar);
                    opar ^= 1;
                    tc_fence_after();
                    const uint64_t b = vdesc + (uint64_t)(vs * (S::vBytes >> 4));
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        mma_f16_ts(elected, t0, t0 + kColP + 8 * k, b + (uint64_t)(k * (2 * S::vLbo >> 4)), idesc_o, i > 0 || k > 0);
                    mma_commit(elected, odone(w));
                    mma_commit(elected, vfree(vs));
                    next_v();
                }
            }
        } else if (warp == 22) {
            // =============================== segments ===============================
            Walk walk;
            walk.cur = cur;
            walk.end = shares.first(blockIdx.x + 1);
            walk.seq = s_seq;
            walk.tile = s_tile;
            walk.at = s_at;
            walk.sequence(p);
            walk.range = range_of(p, walk.len, walk.n, walk.tile);
            int count;
            do {
                batch_sync();
                for (count = 0; count < kSegments && walk.next(p); ++count) {
                    if (lane) continue;
                    Segment &s = s_seg[count];
                    s.tiles = walk.u1 - walk.u0;
                    s.key0 = walk.range.lo + walk.u0 * kKeys;
                    s.see = walk.range.see;
                    s.hi = walk.range.hi;
                    s.seq = walk.seq; s.head = walk.head; s.row0 = walk.row0; s.n = walk.n; s.len = walk.len;
                    s.flat0 = walk.tile * kRows;
                    s.rows = (int)min((long long)kRows, (long long)walk.n * p.G - s.flat0);
                    s.all = walk.u0 == 0 && walk.u1 == walk.range.units - kPairCost;
                    const long long pair_at = walk.at + (long long)walk.head * walk.range.units, pair_end = pair_at + walk.range.units;
                    s.w0 = s.all ? 0 : shares.owner(pair_at + kPairCost);
                    s.w1 = s.all ? 0 : shares.owner(pair_end - 1);
                    s.slot = 2 * blockIdx.x + (walk.u0 == 0 ? 1 : 0);
                }
                if (lane == 0) s_count = count;
                batch_sync();
            } while (count == kSegments);
        }
    }

    // ---- teardown
    if (*err) {                                            // a wait gave up: let what is in flight end
        for (int i = 0; i < 400; ++i) __nanosleep(256);
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && s_err) atomicExch(p.status, s_err);
    if (warp == 20) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

typedef void (*prompt_fn)(const AttendArgs);

}  // namespace prompt

size_t prompt_workspace(int D) { return 2 * (size_t)prompt_grid() * (kPromptRows * (size_t)D + 2 * kPromptRows) * 4; }

int prompt_launch(const AttendArgs &a, int D, bool e4m3, cudaStream_t st) {
    using namespace prompt;
    const prompt_fn kern = D == 64 ? (e4m3 ? prompt_kernel<64, true> : prompt_kernel<64, false>)
                                   : (e4m3 ? prompt_kernel<128, true> : prompt_kernel<128, false>);
    const int smem = D == 64 ? Shape<64>::smem : Shape<128>::smem;
    static jq_contexts done[4];
    JQ_CUDA_TRY(jq_allow_smem(reinterpret_cast<const void *>(kern), smem, done[(D == 128) * 2 + e4m3]));
    kern<<<prompt_grid(), kThreads, smem, st>>>(a);
    return jq_launch_status();
}

}  // namespace jqkv
