// Attention over the 8-bit cache, many query rows per key head (prompts and parts of prompts): tcgen05.
//
// A CTA has 256 rows (query, head of the group) of a key head as two tiles of 128 and walks along the keys in tiles of
// 64.  Four warps turn a tile's codes into fp16 operands in shared memory, once for both row tiles; one warp issues S = Q K^T and O += P V
// (M = 128, N = 64 and N = D, accumulators in tensor memory); four warps for each row tile, a thread per row, turn
// scores into weights, which go back to tensor memory as the A operand of the second product.  Block scales never touch the
// operands: a key block's scale multiplies its columns of S in fp32, a value block's goes into the exponent,
//   t = s ks scale log2(e) + log2(vs),  p = 2^(t - ref),  O = sum p v_code,  l = sum p / vs,  out = O / l,
// and O is only rescaled when a row's maximum has grown by more than 2^8 over its reference (p fits fp16 up to 2^16).
#include "kv_attend.cuh"

namespace jqkv {

using namespace jqta;

namespace prompt {

constexpr int kThreads = 512;      // warps 0-3 and 4-7: the two row tiles, 8-11: codes to operands, 12: matrix instructions
constexpr int kRows = kPromptRows, kKeys = 64;
constexpr int kStages = 4;         // of the rings of key and value operands
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

// (s0, s1) * f + add + shift, two values at once, rounded after each step
__device__ __forceinline__ float2 exponents(uint32_t s0, uint32_t s1, float f, float add, float shift) {
    float2 r;
    asm("{ .reg .b64 s, f, a, t; mov.b64 s, {%2, %3}; mov.b64 f, {%4, %4}; mov.b64 a, {%5, %5}; mov.b64 t, {%6, %6};\n"
        "  fma.rn.f32x2 s, s, f, a; add.rn.f32x2 s, s, t; mov.b64 {%0, %1}, s; }"
        : "=f"(r.x), "=f"(r.y) : "r"(s0), "r"(s1), "f"(f), "f"(add), "f"(shift));
    return r;
}
__device__ __forceinline__ void add2(float2 &a, float2 b) {
    asm("{ .reg .b64 x, y; mov.b64 x, {%0, %1}; mov.b64 y, {%2, %3}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
        : "+f"(a.x), "+f"(a.y) : "f"(b.x), "f"(b.y));
}

// Keys that the rows of a tile see, rounded down to a unit at their beginning.
struct Range {
    int lo, hi, units;
};
__device__ __forceinline__ Range range_of(const AttendArgs &p, int len, int n, int tile) {
    const int first = len - n;
    const int q0 = (int)((long long)tile * kRows / p.G), q1 = (int)min((long long)n - 1, ((long long)(tile + 1) * kRows - 1) / p.G);
    Range r;
    r.hi = max(0, min(len, first + q1 + 1));
    r.lo = p.window > 0 ? max(0, first + q0 - p.window + 1) : 0;
    r.lo = min(r.lo, r.hi) & ~(kKeys - 1);
    r.units = max(1, (r.hi - r.lo + kKeys - 1) / kKeys);
    return r;
}
__device__ __forceinline__ int tiles_of(const AttendArgs &p, int n) { return (int)(((long long)n * p.G + kRows - 1) / kRows); }

// The segments of a CTA: units in the order (sequence, row tile, key head, unit), cut evenly.
struct Walk {
    long long cur, end, at;        // at: first unit of (seq, tile)
    int seq, tile, n, len, row0, tiles;
    Range range;
    // of the segment
    int head, u0, u1;
    __device__ __forceinline__ void sequence(const AttendArgs &p) {
        n = p.b.count(seq, row0);
        len = p.b.length(seq);
        tiles = tiles_of(p, n);
    }
    __device__ __forceinline__ bool next(const AttendArgs &p) {
        if (cur >= end) return false;
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
        head = (int)(in / range.units);
        u0 = (int)(in % range.units);
        u1 = (int)min((long long)range.units, u0 + (end - cur));
        cur += u1 - u0;
        return true;
    }
    __device__ __forceinline__ int rows(const AttendArgs &p) const { return (int)min((long long)kRows, (long long)n * p.G - (long long)tile * kRows); }
    __device__ __forceinline__ int key0() const { return range.lo + u0 * kKeys; }
};

template <int D, bool E4M3>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ AttendArgs p) {
    using S = Shape<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[4 * kStages + 2 * 5 + kScaleSlots];
    __shared__ float s_scales[kScaleSlots][4][4];            // [.][group]: factor of the scores (negative: not there), log2(vs), 1 / vs
    __shared__ long long s_sum[8], s_at;
    __shared__ int s_err, s_seq, s_tile, s_last;
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
    auto scales_full = [&](int s) { return b0 + 8 * (4 * kStages + 10 + s); };

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
            mbar_init(kfree(s), 1);
            mbar_init(vfree(s), 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(qfull(w), 4);
            mbar_init(sfull(w), 1);
            mbar_init(sfree(w), 4);
            mbar_init(pfull(w), 4);
            mbar_init(odone(w), 1);
        }
        for (int s = 0; s < kScaleSlots; ++s) mbar_init(scales_full(s), 4);
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
    const long long fit = (total + p.least - 1) / p.least;
    const int W = fit < (long long)gridDim.x ? (int)fit : (int)gridDim.x;
    if ((int)blockIdx.x >= W) return;
    Walk walk;
    walk.cur = total * blockIdx.x / W;
    walk.end = total * (blockIdx.x + 1) / W;
    if (tid < 256 && walk.cur >= before && walk.cur < before + mine) {
        long long at = before;
        for (int i = 0; i < my_seqs; ++i) {
            int row0;
            const int n = p.b.count(my_seq + i, row0), len = p.b.length(my_seq + i), tiles = tiles_of(p, n);
            for (int t = my_tile; t < min(my_tiles, tiles); ++t) {
                const long long u = (long long)range_of(p, len, n, t).units * p.H;
                if (walk.cur >= at && walk.cur < at + u) {
                    s_seq = my_seq + i;
                    s_tile = t;
                    s_at = at;
                }
                at += u;
            }
        }
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    walk.seq = s_seq;
    walk.tile = s_tile;
    walk.at = s_at;
    walk.sequence(p);
    walk.range = range_of(p, walk.len, walk.n, walk.tile);
    volatile int *err = &s_err;
    auto wait = [&](uint32_t bar, uint32_t parity) {          // (converged again behind it: what follows is often the whole warp's)
        mbar_wait(bar, parity, err);
        __syncwarp();
    };
    unsigned char *const kring = smem, *const vring = smem + kStages * S::kKBytes, *const qmem = vring + kStages * S::vBytes;

    // Registers: 512 x 128 at launch = 256 x 160 + 128 x 112 + 128 x 80
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        // =============================== scores to weights: a thread per row ===============================
        const int w = warp >> 2, r = tid & 127;
        const uint32_t mine_t = tmem + w * kColTile + ((uint32_t)(warp & 3) << 21);      // this warp's 32 lanes of its tile
        uint32_t it = 0;                                   // tiles of this row tile so far
        int slot = 0;                                      // of the scales
        uint32_t slot_par = 0;
        while (walk.next(p)) {
            const int tiles = walk.u1 - walk.u0, rows = walk.rows(p);
            const bool active = w == 0 || rows > 128;
            const long long flat = (long long)walk.tile * kRows + w * 128 + r;           // row among the sequence's
            const bool there = w * 128 + r < rows;
            const int j = there ? (int)(flat / p.G) : 0, hq = walk.head * p.G + (there ? (int)(flat % p.G) : 0);
            const int pos = there ? walk.len - walk.n + j : -1;
            float ref = -INFINITY, l = 0.f, qs = 0.f;
            if (active) {
                // the query row, divided by a power of two that brings it into fp16's range
                const unsigned short *at = reinterpret_cast<const unsigned short *>(p.q) + (walk.row0 + j) * p.st + hq * p.sh;
                const bool vec = (reinterpret_cast<uintptr_t>(at) & 15u) == 0;
                auto load = [&](int c) -> uint4 {
                    uint4 u = make_uint4(0, 0, 0, 0);
                    if (there) {
                        if (vec) {
                            u = reinterpret_cast<const uint4 *>(at)[c];
                        } else {
                            unsigned short *e = reinterpret_cast<unsigned short *>(&u);
#pragma unroll
                            for (int k = 0; k < 8; ++k) e[k] = at[c * 8 + k];
                        }
                    }
                    return u;
                };
                auto value = [&](uint32_t x, int hi_half) -> float {
                    const unsigned short u = (unsigned short)(hi_half ? x >> 16 : x & 0xffffu);
                    return p.dtype == JQ_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float((uint32_t)u << 16);
                };
                float amax = 0.f;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const uint4 u = load(c);
                    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(fabsf(value(x[k], 0)), fabsf(value(x[k], 1))));
                }
                const int e = act_exponent(amax, false);
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                qs = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int c4 = 0; c4 < D / 32; ++c4) {
                    uint32_t h[16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint4 u = load(c4 * 4 + c);
                        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) h[c * 4 + k] = pack_h2(value(x[k], 0) * down, value(x[k], 1) * down);
                    }
                    if (c4 * 32 < kQTmem) {
                        tmem_st16(mine_t + kColQ + c4 * 16, h);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint4 *>(qmem + w * S::qBytes + ((c4 - kQTmem / 32) * 4 + c) * 2048 + r * 16) =
                                make_uint4(h[c * 4], h[c * 4 + 1], h[c * 4 + 2], h[c * 4 + 3]);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull(w));
            }
            int key = walk.key0();
            for (int i = 0; i < tiles; ++i, key += kKeys) {
                if (active) {
                    wait(scales_full(slot), slot_par);
                    wait(sfull(w), it & 1);
                    tc_fence_after();
                    uint32_t s[64];
                    tmem_ld32(mine_t + kColS, *reinterpret_cast<uint32_t(*)[32]>(s));
                    tmem_ld32(mine_t + kColS + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sfree(w));
                    float4 sc[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) sc[n] = *reinterpret_cast<const float4 *>(s_scales[slot][n]);
                    const int last = pos - key, first = p.window > 0 ? last - p.window + 1 : -1;     // columns that the row sees
                    const bool edge = last < kKeys - 1 || first > 0 || sc[0].x < 0.f || sc[1].x < 0.f || sc[2].x < 0.f || sc[3].x < 0.f;
                    if (__any_sync(0xffffffffu, edge)) {
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (c > last || c < first || sc[c >> 4].x < 0.f) s[c] = 0xff800000u;
                    }
                    float top = -INFINITY, f[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        float m = __uint_as_float(s[16 * n]);
#pragma unroll
                        for (int c = 1; c < 16; ++c) m = fmaxf(m, __uint_as_float(s[16 * n + c]));
                        f[n] = fabsf(sc[n].x) * qs;
                        top = fmaxf(top, fmaf(m, f[n], sc[n].y));
                    }
                    if (i == 0) {
                        ref = top;
                    } else if (__any_sync(0xffffffffu, top > ref + 8.f)) {
                        const float to = top > ref + 8.f ? top : ref;
                        const float a = to == -INFINITY ? 1.f : ex2(ref - to);
                        ref = to;
                        l *= a;
                        wait(odone(w), (it & 1) ^ 1);
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(mine_t + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * a);
                            tmem_st16(mine_t + c * 32, *reinterpret_cast<uint32_t(*)[16]>(o));
                            tmem_st16(mine_t + c * 32 + 16, *reinterpret_cast<uint32_t(*)[16]>(o + 16));
                        }
                        tmem_wait_st();
                    }
                    const float base = ref == -INFINITY ? 0.f : ref;
                    wait(odone(w), (it & 1) ^ 1);                        // the weights of the tile before have been used
                    uint32_t h[16];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        // (the exponent as the maximum was formed, then the difference: both at once would leave the rounding of
                        // a large exponent in the weight)
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            const float2 e = exponents(s[16 * n + c], s[16 * n + c + 1], f[n], sc[n].y, -base);
                            const float2 a = make_float2(ex2(e.x), ex2(e.y));
                            add2(sum, a);
                            h[8 * (n & 1) + c / 2] = pack_h2(a.x, a.y);
                        }
                        l = fmaf(sum.x + sum.y, sc[n].z, l);
                        if (n & 1) tmem_st16(mine_t + kColP + 8 * (n - 1), h);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pfull(w));
                    ++it;
                }
                if (++slot == kScaleSlots) { slot = 0; slot_par ^= 1; }
            }
            // ---- outputs, or a part of them
            const bool all = walk.u0 == 0 && walk.u1 == walk.range.units;
            const long long pair_at = walk.at + (long long)walk.head * walk.range.units, pair_end = pair_at + walk.range.units;
            const int w0 = all ? 0 : (int)(((pair_at + 1) * W - 1) / total), w1 = all ? 0 : (int)((pair_end * W - 1) / total);
            float *part = p.parts + (size_t)(2 * blockIdx.x + (walk.u0 == 0 ? 1 : 0)) * S::part;
            const size_t out_at = ((size_t)(walk.row0 + j) * p.H * p.G + hq) * D;
            if (active) {
                wait(odone(w), (it & 1) ^ 1);
                tc_fence_after();
                const float inv = inverse(l);
                if (all && there && p.lse) p.lse[out_at / D] = lse_of(ref, l);
                if (!all && there) {
                    part[kRows * D + w * 128 + r] = ref;
                    part[kRows * D + kRows + w * 128 + r] = l;
                }
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(mine_t + c * 32, o);
                    tmem_wait_ld();
                    if (there) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        float v[8];
#pragma unroll
                        for (int x = 0; x < 8; ++x) v[x] = __uint_as_float(o[k + x]);
                        if (all) {
                            store8(p, out_at + c * 32 + k, v, inv);
                        } else {
                            float4 *dst = reinterpret_cast<float4 *>(part + (size_t)(w * 128 + r) * D + c * 32 + k);
                            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                        }
                    }
                    }
                    __syncwarp();
                }
                tc_fence_before();
            }
            if (!all) {
                // the last of the pair's CTAs to get here adds the parts, in their order
                __threadfence();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (tid == 0) {
                    const int n = atomicAdd(p.counters + w0, 1);
                    s_last = n == w1 - w0;
                    if (s_last) p.counters[w0] = 0;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (s_last) {
                    __threadfence();
                    for (int e = tid; e < rows * (D / 4); e += 256) {
                        const int row = e / (D / 4), d = e % (D / 4) * 4;
                        float m = -INFINITY, lsum = 0.f;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int k = w0; k <= w1; ++k) {
                            const float *x = p.parts + (size_t)(2 * k + (k == w0 ? 1 : 0)) * S::part;
                            add_part(m, lsum, v, __ldcg(x + kRows * D + row), __ldcg(x + kRows * D + kRows + row),
                                     __ldcg(reinterpret_cast<const float4 *>(x + (size_t)row * D + d)));
                        }
                        const long long fr = (long long)walk.tile * kRows + row;
                        const size_t o = ((size_t)(walk.row0 + fr / p.G) * p.H * p.G + walk.head * p.G + fr % p.G) * D;
                        store4(p, o + d, v, inverse(lsum));
                        if (d == 0 && p.lse) p.lse[o / D] = lse_of(m, lsum);
                    }
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");           // (s_last is read before the next segment writes it)
            }
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // =============================== codes to operands: a warp per 16 keys of a tile ===============================
        const int cw = warp - 8, g = lane >> 2, t = lane & 3;
        constexpr int C = D / 32;
        int st = 0, slot = 0;
        uint32_t par = 1;                                  // (the first round finds every stage free)
        const uint32_t none = E4M3 ? 0u : 0x80808080u;     // code of 0
        while (walk.next(p)) {
            const int tiles = walk.u1 - walk.u0, key0 = walk.key0() + 16 * cw;
            int id = -1;
            float kc = -1.f, vl = 0.f, vi = 1.f;
            auto look_up = [&](int first) {                // lane l: block and scales of tile first + l
                const int k = key0 + (first + lane) * kKeys;
                id = -1;
                if (first + lane < tiles && k < walk.range.hi) id = p.b.block(walk.seq, k);
                kc = -1.f;
                vl = 0.f;
                vi = 1.f;
                if (id >= 0) {
                    const size_t at = (size_t)id * p.H + walk.head;
                    const float v = p.vs[at];
                    kc = p.ks[at] * p.scale;
                    vl = log2f(v);
                    vi = __fdividef(1.f, v);
                }
            };
            uint4 kr[C], vr[C];
            auto load = [&](const uint8_t *codes, int tile, uint4 (&x)[C]) {     // (ids of the 32 tiles that `tile` is one of)
                const int b = __shfl_sync(0xffffffffu, id, tile & 31);
                const int k = key0 + tile * kKeys;
                const uint4 *at = reinterpret_cast<const uint4 *>(codes + (((size_t)max(b, 0) * p.H + walk.head) * p.b.T + k % p.b.T) * D) + lane;
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
                if (lane == 0) {
                    *reinterpret_cast<float4 *>(s_scales[slot][cw]) = make_float4(kc_i, vl_i, vi_i, 0.f);
                    mbar_arrive(scales_full(slot));
                }
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
                    const int left = walk.len - (key0 + i * kKeys + 4 * t);
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
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 12) {
        // =============================== matrix instructions ===============================
        // (the warp runs converged, see mma_f16_ts)
        const uint32_t elected = elect_one();
        const uint64_t kdesc = smem_desc(smem_u32(kring), S::kLbo, 128), vdesc = smem_desc(smem_u32(vring), S::vLbo, 128),
                       qdesc = smem_desc(smem_u32(qmem), 2048, 128);
        constexpr uint32_t idesc_s = idesc_f16(128, kKeys), idesc_o = idesc_f16(128, D);
        int ks = 0, vs = 0;
        uint32_t kpar = 0, vpar = 0, qpar[2] = {0, 0}, it[2] = {0, 0};          // it: scores of the row tile so far
        auto scores = [&](int w) {
            wait(sfree(w), (it[w] & 1) ^ 1);
            tc_fence_after();
            const uint32_t t0 = tmem + w * kColTile;
            const uint64_t b = kdesc + (uint64_t)(ks * (S::kKBytes >> 4));
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                if (k < kQTmem / 16) mma_f16_ts(elected, t0 + kColS, t0 + kColQ + 8 * k, b + (uint64_t)(k * (2 * S::kLbo >> 4)), idesc_s, k > 0);
                else mma_f16_ss(elected, t0 + kColS, qdesc + (uint64_t)((w * S::qBytes + (k - kQTmem / 16) * 4096) >> 4),
                                b + (uint64_t)(k * (2 * S::kLbo >> 4)), idesc_s, 1);
            }
            mma_commit(elected, sfull(w));
            ++it[w];
        };
        uint32_t ot[2] = {0, 0};                           // outputs of the row tile so far
        while (walk.next(p)) {
            const int tiles = walk.u1 - walk.u0, both = walk.rows(p) > 128 ? 2 : 1;
            for (int w = 0; w < both; ++w) {
                wait(qfull(w), qpar[w]);
                qpar[w] ^= 1;
            }
            tc_fence_after();
            auto step = [&](int i, int w) {                // scores of tile i + 1, then outputs of tile i
                if (i + 1 < tiles) {
                    if (w == 0) wait(kfull(ks), kpar);
                    scores(w);
                    if (w == both - 1) {
                        mma_commit(elected, kfree(ks));
                        if (++ks == kStages) { ks = 0; kpar ^= 1; }
                    }
                }
                if (i >= 0) {
                    if (w == 0) wait(vfull(vs), vpar);
                    wait(pfull(w), ot[w] & 1);
                    ++ot[w];
                    tc_fence_after();
                    const uint32_t t0 = tmem + w * kColTile;
                    const uint64_t b = vdesc + (uint64_t)(vs * (S::vBytes >> 4));
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        mma_f16_ts(elected, t0, t0 + kColP + 8 * k, b + (uint64_t)(k * (2 * S::vLbo >> 4)), idesc_o, i > 0 || k > 0);
                    mma_commit(elected, odone(w));
                    if (w == both - 1) {
                        mma_commit(elected, vfree(vs));
                        if (++vs == kStages) { vs = 0; vpar ^= 1; }
                    }
                }
            };
            for (int i = -1; i < tiles; ++i)
                for (int w = 0; w < both; ++w) step(i, w);
        }
        }
    }

    // ---- teardown
    if (*err) {                                            // a wait gave up: let what is in flight end
        for (int i = 0; i < 400; ++i) __nanosleep(256);
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && s_err) atomicExch(p.status, s_err);
    if (warp == 12) {
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
