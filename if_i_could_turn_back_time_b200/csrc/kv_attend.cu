// Attention over the 8-bit cache, few query rows per key head (single tokens, drafts).
//
// Bound by reading the cache: 64 sequences of 257 to 8191 tokens, 8 key heads of 128, 556 MB: 104 us, 5.3 TB/s (107 under the power cap); one of 131071, 269 MB: 62 us.
// One row of 517 tokens and 32 heads takes 8 us, a chain of global latencies: lengths, table, copies, the join of the parts.
#include "kv_attend.cuh"

namespace jqkv {

using namespace jqta;

constexpr int kNear = 16;          // units: how far a boundary between CTAs moves to a pair's begin or end, at most half a CTA's share (see snap)
constexpr int kUnit = 64;          // keys: what work is dealt out in
constexpr float kLift = 14.f;      // a row's reference lies 2^14 below its largest weight, so that fp16 weights have eleven bits down to 2^-28 of it
constexpr int kRing = 16384;       // bytes of a warp's ring: two stages of 32 keys at D = 128, three CTAs on an SM

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Warps of a CTA: four, two or three CTAs on an SM, so that one's beginning and end fall into the others' loops; or all of an SM's.
__host__ __device__ constexpr int warps_of(int NT, bool wide) { return wide ? (NT > 2 ? 8 : 12) : 4; }

// A matrix of 8 x 8 fp16 values, two of a row in a lane (row lane / 4), the other way round.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// A sequence's share of the work: row tiles x key heads pairs of `units` units each, pairs in the order (head, tile).
struct Share {
    int row0, n, len, see, lo, units, tiles;       // see: first key that any row sees; lo: the unit that it lies in
    long long total;
};
template <int ROWS>
__device__ __forceinline__ Share share_of(const AttendArgs &p, int i) {
    Share s;
    s.n = p.b.count(i, s.row0);
    s.len = p.b.length(i);
    s.see = first_seen(p, s.len - s.n);
    s.lo = s.see & ~(kUnit - 1);
    s.units = max(1, (s.len - s.lo + kUnit - 1) / kUnit);      // (a row that sees nothing has its zeros written too)
    s.tiles = (int)(((long long)s.n * p.G + ROWS - 1) / ROWS);
    s.total = (long long)s.tiles * p.H * s.units;
    return s;
}

// The parts of a pair, of the CTAs w0 .. w1, added in their order; outputs.  (Not inlined: its registers are not the main loop's.  Forming all
// factors first, so that the loads of the sums wait for nothing, took as long for 3 to 55 parts.)
template <int D, int TR, int THREADS>
__device__ __noinline__ void add_parts(const AttendArgs &p, int w0, int w1, int rows, int r0, int row0, int h) {
    constexpr int kPart = TR * D + 2 * TR;
    for (int e = threadIdx.x; e < rows * (D / 4); e += THREADS) {
        const int r = e / (D / 4), d = e % (D / 4) * 4, fr = r0 + r;
        float m = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int w = w0; w <= w1; ++w) {
            const float *x = p.parts + (size_t)(2 * w + (w == w0 ? 1 : 0)) * kPart;
            add_part(m, l, v, __ldcg(x + TR * D + r), __ldcg(x + TR * D + TR + r), __ldcg(reinterpret_cast<const float4 *>(x + r * D + d)));
        }
        const size_t at = ((size_t)(row0 + fr / p.G) * p.H * p.G + h * p.G + fr % p.G) * D + d;
        store4(p, at, v, inverse(l));
        if (d == 0 && p.lse) p.lse[at / D] = lse_of(m, l);
    }
}

// NT: tiles of 8 query rows (query, head of the group).  Both products have the cache as their 16-row operand, so that 8 query rows cost
// one instruction for 16 keys x 16 values: S^T = K Q^T, O^T = V^T P^T.  A lane has the scores of the keys (g, 0) and (g, 1) of a
// group (see kv.cuh) for the rows 2t and 2t + 1; packed to fp16 and transposed by movmatrix they are the second product's B operand.
template <int D, bool E4M3, int NT, bool WIDE>
__global__ void __launch_bounds__(warps_of(NT, WIDE) * 32, WIDE ? 1 : (NT > 2 ? 2 : 3)) attend_kernel(const __grid_constant__ AttendArgs p) {
    constexpr int kWarps = warps_of(NT, WIDE);                 // each takes every kWarps-th stage of a segment
    constexpr int C = D / 32;                                  // chunks of a group
    constexpr int KEYS = 32, NG = KEYS / 16;                   // keys and groups of a stage
    constexpr int kStageBytes = KEYS * D * 2;
    constexpr int NS = kRing / kStageBytes;                    // stages of a warp's ring
    constexpr int TR = NT * 8;                                 // rows of a tile
    constexpr int kPart = TR * D + 2 * TR;                     // floats of a part
    constexpr int kPitch = D + 4;                              // floats of a row on its way to the other warps: rows 2t, 2t + 2, .. in different banks
    static_assert(TR * kPitch * 4 <= kRing || NT == 4, "a warp's sums take the place of its ring");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[kWarps * NS];
    __shared__ int s_err, s_seq, s_last;
    __shared__ long long s_sum[kWarps], s_off;
    __shared__ Share s_share;
    __shared__ float s_m[kWarps][TR], s_l[kWarps][TR];

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, tq = lane & 3;
    constexpr int kOwn = TR * kPitch * 4 > kRing ? TR * kPitch * 4 : kRing;
    unsigned char *const ring = smem + warp * kOwn;
    const uint32_t ring_u = smem_u32(ring), bar0 = smem_u32(&bars[warp * NS]);
    if (lane == 0)
        for (int s = 0; s < NS; ++s) mbar_init(bar0 + 8 * s, 1);
    if (tid == 0) s_err = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();

    // ---- this CTA's units: [lo, hi) of all, the same number for every CTA up to one
    const int per = (p.b.S + kWarps * 32 - 1) / (kWarps * 32), i0 = min(p.b.S, tid * per), i1 = min(p.b.S, i0 + per);
    long long mine = 0;
    for (int i = i0; i < i1; ++i) mine += share_of<TR>(p, i).total;
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) before += total - mine;
        total += s_sum[w];
    }
    if (total == 0) return;
    const long long fit = quotient(total + p.least - 1, p.least);
    const int W = fit < (long long)gridDim.x ? (int)fit : (int)gridDim.x;
    if ((int)blockIdx.x >= W) return;
    const Shares shares(total, W);
    const long long lo = shares.first(blockIdx.x);
    long long cur = lo;
    const long long near = shares.base > 2 * kNear ? kNear : shares.base / 2;
    const long long hi = shares.first(blockIdx.x + 1);
    if (cur >= before && cur < before + mine) {                // (one thread's sequences hold the first unit)
        long long at = before;
        for (int i = i0; i < i1; ++i) {
            const Share s = share_of<TR>(p, i);
            if (cur < at + s.total) {
                s_seq = i;
                s_off = at;
                s_share = s;
                break;
            }
            at += s.total;
        }
    }
    __syncthreads();
    int seq = s_seq;
    long long seq_at = s_off;
    Share sh = s_share;

    uint32_t phases = 0;                                       // parity of each stage's next completion
    while (cur < hi) {
        while (cur >= seq_at + sh.total) {
            seq_at += sh.total;
            sh = share_of<TR>(p, ++seq);
        }
        const int pair = (int)quotient(cur - seq_at, sh.units);
        const long long pair_at = seq_at + (long long)pair * sh.units, pair_end = pair_at + sh.units;
        // A boundary between two CTAs that is near a pair's begin or end is taken to lie there: a few units more for one of them are
        // less than a further segment (one row of 517 tokens, 32 heads: 9.7 us, 15.9 with boundaries as they fall; 64 sequences of
        // 257 to 8191 tokens, 8 key heads: 100 and 107).
        auto snap = [&](long long b) {
            const long long off = b - pair_at, rest = pair_end - b;
            return off <= near && off <= rest ? pair_at : (rest <= near ? pair_end : b);
        };
        const long long from = cur == lo ? snap(cur) : cur, to = hi < pair_end ? snap(hi) : pair_end;
        cur = pair_end;
        if (to <= from) continue;
        const int u0 = (int)(from - pair_at), u1 = (int)(to - pair_at);
        const int h = sh.tiles == 1 ? pair : pair / sh.tiles, tile = sh.tiles == 1 ? 0 : pair % sh.tiles;
        const int k0 = sh.lo + u0 * kUnit, k1 = min(sh.len, sh.lo + u1 * kUnit);
        const int stages = k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0;
        const int own = stages > warp ? (stages - warp + kWarps - 1) / kWarps : 0;      // stages of this warp
        const int r0 = tile * TR, rows = min(TR, sh.n * p.G - r0);

        // ---- the warp's stages, 32 of them at a time: lane l has the blocks and scales of the l-th
        int id[NG];
        float kc[NG], vl[NG], vi[NG];
        auto look_up = [&](int first) {
            const int st = first + lane;
            const int key = k0 + (warp + st * kWarps) * KEYS;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                id[n] = -1;
                // (16 keys that nobody sees are not looked at: their block may be another sequence's by now)
                if (st < own && key + 16 * n < k1 && key + 16 * n + 16 > sh.see) id[n] = p.b.block(seq, key + 16 * n);
            }
        };
        auto scales = [&]() {
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const size_t at = (size_t)max(id[n], 0) * p.H + h;
                const float v = id[n] >= 0 ? p.vs[at] : 1.f;
                kc[n] = id[n] >= 0 ? p.ks[at] : 0.f;
                vl[n] = log2f(v);
                vi[n] = __fdividef(1.f, v);
            }
        };
        auto issue = [&](int st, int slot) {                   // all lanes; stage `st` of the warp, within the 32 looked up
            int ids[NG];
#pragma unroll
            for (int n = 0; n < NG; ++n) ids[n] = __shfl_sync(0xffffffffu, id[n], st & 31);
            if (lane == 0) {
                const int key = k0 + (warp + st * kWarps) * KEYS;
                const uint32_t bar = bar0 + 8 * slot, dst = ring_u + slot * kStageBytes;
                uint32_t bytes = 0;
#pragma unroll
                for (int n = 0; n < NG; ++n) bytes += ids[n] >= 0 ? 32 * D : 0;
                mbar_expect_tx(bar, bytes);
                if (ids[0] >= 0 && ids[1] >= 0 && p.b.T >= KEYS) {
                    const size_t at = (((size_t)ids[0] * p.H + h) * p.b.T + (key & (p.b.T - 1))) * D;
                    bulk_g2s(dst, p.keys + at, KEYS * D, bar);
                    bulk_g2s(dst + KEYS * D, p.values + at, KEYS * D, bar);
                } else {
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        if (ids[n] < 0) continue;
                        const size_t at = (((size_t)ids[n] * p.H + h) * p.b.T + ((key + 16 * n) & (p.b.T - 1))) * D;
                        bulk_g2s(dst + n * 16 * D, p.keys + at, 16 * D, bar);
                        bulk_g2s(dst + KEYS * D + n * 16 * D, p.values + at, 16 * D, bar);
                    }
                }
            }
        };
        look_up(0);
        // ---- queries, row g of each tile as the B operand, divided by a power of two that brings the row into fp16's range
        uint4 raw[NT][C];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g, fr = r0 + (r < rows ? r : 0);                    // (a row that is not there reads the tile's first)
            const unsigned short *at = reinterpret_cast<const unsigned short *>(p.q) + (sh.row0 + fr / p.G) * p.st + (h * p.G + fr % p.G) * p.sh + tq * 8;
            if ((p.st | p.sh) % 8 == 0 && (reinterpret_cast<uintptr_t>(p.q) & 15u) == 0) {
#pragma unroll
                for (int c = 0; c < C; ++c) raw[nt][c] = __ldg(reinterpret_cast<const uint4 *>(at + c * 32));
            } else {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    uint32_t x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = at[c * 32 + 2 * k] | (uint32_t)at[c * 32 + 2 * k + 1] << 16;
                    raw[nt][c] = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (s < own) issue(s, s);
        scales();
        uint32_t qb[NT][C][2][2];
        float qs[NT][2];                                       // what the scores of the rows 2t and 2t + 1 are multiplied by
        int pos[NT][2];                                        // their positions; -1: no such row
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            auto value = [&](uint32_t w, int hi_half) -> float {
                const unsigned short u = (unsigned short)(hi_half ? w >> 16 : w & 0xffffu);
                return p.dtype == JQ_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float((uint32_t)u << 16);
            };
            float amax = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t w[4] = {raw[nt][c].x, raw[nt][c].y, raw[nt][c].z, raw[nt][c].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(fabsf(value(w[k], 0)), fabsf(value(w[k], 1))));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int e = query_exponent(amax);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t w[4] = {raw[nt][c].x, raw[nt][c].y, raw[nt][c].z, raw[nt][c].w};
#pragma unroll
                for (int k = 0; k < 4; ++k)                    // word k: values 2k, 2k + 1 = step k / 2, register k % 2
                    qb[nt][c][k >> 1][k & 1] = pack_h2(value(w[k], 0) * down, value(w[k], 1) * down);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = nt * 8 + 2 * tq + k, ee = __shfl_sync(0xffffffffu, e, (2 * tq + k) * 4);
                qs[nt][k] = __uint_as_float((uint32_t)(127 + ee) << 23) * p.scale;
                pos[nt][k] = r < rows ? sh.len - sh.n + (r0 + r) / p.G : -1;
            }
        }

        float o[NT][D / 16][4], M[NT][2], l[NT][2];            // o: values 16 i + g and 16 i + g + 8 of the rows 2t, 2t + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            M[nt][0] = M[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) o[nt][n][0] = o[nt][n][1] = o[nt][n][2] = o[nt][n][3] = 0.f;
        }
        // the queries' least and largest positions: keys between them and the window's edges are looked at one by one
        const int pos_first = sh.len - sh.n + r0 / p.G, pos_last = sh.len - sh.n + (r0 + rows - 1) / p.G;

        int slot = 0;
        for (int st = 0; st < own; ++st) {
            const int sl = st & 31;
            const int key = k0 + (warp + st * kWarps) * KEYS;
            mbar_wait(bar0 + 8 * slot, phases >> slot & 1, &s_err);
            __syncwarp();
            phases ^= 1u << slot;
            const uint32_t base = ring_u + slot * kStageBytes + lane * 16;
            float kcs[NG], vls[NG], vis[NG];
            bool there[NG];
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                kcs[n] = __shfl_sync(0xffffffffu, kc[n], sl);
                vls[n] = __shfl_sync(0xffffffffu, vl[n], sl);
                vis[n] = __shfl_sync(0xffffffffu, vi[n], sl);
                there[n] = __shfl_sync(0xffffffffu, id[n], sl) >= 0;
            }
            float s[NT][NG][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int n = 0; n < NG; ++n) s[nt][n][0] = s[nt][n][1] = s[nt][n][2] = s[nt][n][3] = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    const uint4 w = lds128(base + n * 16 * D + c * 512);
                    uint32_t a[2][4];                          // the two steps of 16 values
                    codes_to_h4<E4M3>(w.x, a[0][0], a[0][2]);
                    codes_to_h4<E4M3>(w.y, a[1][0], a[1][2]);
                    codes_to_h4<E4M3>(w.z, a[0][1], a[0][3]);
                    codes_to_h4<E4M3>(w.w, a[1][1], a[1][3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816(s[nt][n], a[0], qb[nt][c][0][0], qb[nt][c][0][1]);
                        mma16816(s[nt][n], a[1], qb[nt][c][1][0], qb[nt][c][1][1]);
                    }
                }
            // t = log2(weight of the key times its block's value scale); the sums are formed relative to M, the largest t less kLift
            const bool masked = key + KEYS - 1 > pos_first || (p.window > 0 && key <= pos_last - p.window) || !there[0] || !there[NG - 1];
            uint32_t pb[NT][NG][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float alpha[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {                  // row 2t + k; element 2 j + k: key (g, j)
                    float m = -INFINITY;
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        const float f = kcs[n] * qs[nt][k];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float &t = s[nt][n][2 * j + k];
                            t = fmaf(t, f, vls[n]);
                            if (masked) {
                                const int kp = key + n * 16 + 4 * (g >> 1) + (g & 1) + 2 * j;
                                if (kp > pos[nt][k] || (p.window > 0 && kp <= pos[nt][k] - p.window) || !there[n]) t = -INFINITY;
                            }
                            m = fmaxf(m, t);
                        }
                    }
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(M[nt][k], m - kLift);
                    const float ref = m == -INFINITY ? 0.f : m;          // (nothing seen yet: every weight is 0)
                    alpha[k] = ex2(M[nt][k] - ref);
                    M[nt][k] = m;
                    float sum = 0.f;
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        float &t0 = s[nt][n][k], &t1 = s[nt][n][2 + k];
                        t0 = ex2(t0 - ref);
                        t1 = ex2(t1 - ref);
                        sum = fmaf(t0 + t1, vis[n], sum);
                    }
                    l[nt][k] = fmaf(l[nt][k], alpha[k], sum);
                }
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) pb[nt][n][j] = transpose8x8(pack_h2(s[nt][n][2 * j], s[nt][n][2 * j + 1]));
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) {
                        o[nt][n][0] *= alpha[0];
                        o[nt][n][1] *= alpha[1];
                        o[nt][n][2] *= alpha[0];
                        o[nt][n][3] *= alpha[1];
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                // e4m3 has a NaN, and places behind a sequence's end, or of a block that is not there, may hold anything
                uint32_t keep = 0xffffffffu;
                if (E4M3) {
                    const int left = there[n] ? sh.len - (key + n * 16 + 4 * tq) : 0;
                    keep = left >= 4 ? 0xffffffffu : (left <= 0 ? 0u : (1u << 8 * left) - 1u);
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    uint4 w = lds128(base + KEYS * D + n * 16 * D + c * 512);
                    if (E4M3) { w.x &= keep; w.y &= keep; w.z &= keep; w.w &= keep; }
                    uint32_t a[2][4];                          // values g, g + 8 and g + 16, g + 24 of the chunk
                    codes_to_h4<E4M3>(w.x, a[0][0], a[0][2]);
                    codes_to_h4<E4M3>(w.y, a[0][1], a[0][3]);
                    codes_to_h4<E4M3>(w.z, a[1][0], a[1][2]);
                    codes_to_h4<E4M3>(w.w, a[1][1], a[1][3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816(o[nt][c * 2], a[0], pb[nt][n][0], pb[nt][n][1]);
                        mma16816(o[nt][c * 2 + 1], a[1], pb[nt][n][0], pb[nt][n][1]);
                    }
                }
            }
            __syncwarp();                                      // every lane has read the stage
            if (sl == 31 && st + 1 < own) {                    // (the stages in flight keep their codes; their scales are looked up anew)
                look_up(st + 1);
                scales();
            }
            if (st + NS < own) {
                if ((st + NS) / 32 == (st + 1) / 32) {
                    issue(st + NS, slot);
                } else {                                       // its block lies in the next 32: looked up for it alone
                    int keep_id[NG];
#pragma unroll
                    for (int n = 0; n < NG; ++n) keep_id[n] = id[n];
                    look_up((st + NS) & ~31);
                    issue(st + NS, slot);
#pragma unroll
                    for (int n = 0; n < NG; ++n) id[n] = keep_id[n];
                }
            }
            if (++slot == NS) slot = 0;
        }
        // (stages are dealt to slots from slot 0 in every segment; all copies of this one have been waited for)

        // ---- the warps' sums become one
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float v = l[nt][k];
                v += __shfl_xor_sync(0xffffffffu, v, 4);
                v += __shfl_xor_sync(0xffffffffu, v, 8);
                v += __shfl_xor_sync(0xffffffffu, v, 16);
                const int r = nt * 8 + 2 * tq + k;
                if (g == 0) {
                    s_m[warp][r] = M[nt][k];
                    s_l[warp][r] = v;
                }
                float *dst = reinterpret_cast<float *>(ring) + r * kPitch + g;
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    dst[n * 16] = o[nt][n][k];
                    dst[n * 16 + 8] = o[nt][n][2 + k];
                }
            }
        __syncthreads();
        const bool all = u0 == 0 && u1 == sh.units;
        int w0 = 0, w1 = 0;                                    // CTAs that have a part of the pair
        if (!all) {
            w0 = shares.owner(pair_at);
            w1 = shares.owner(pair_end - 1);
            if (w0 < w1 && snap(shares.first(w0 + 1)) == pair_at) ++w0;
            if (w0 < w1 && snap(shares.first(w1)) == pair_end) --w1;
        }
        float *part = p.parts + (size_t)(2 * blockIdx.x + (u0 == 0 ? 1 : 0)) * kPart;
        auto finish = [&](int r, int d, float4 v, float m, float lsum) {      // outputs of four values of a row
            const int fr = r0 + r;
            const size_t at = ((size_t)(sh.row0 + fr / p.G) * p.H * p.G + h * p.G + fr % p.G) * D + d;
            store4(p, at, v, inverse(lsum));
            if (d == 0 && p.lse) p.lse[at / D] = lse_of(m, lsum);
        };
        for (int e = tid; e < rows * (D / 4); e += kWarps * 32) {
            const int r = e / (D / 4), d = e % (D / 4) * 4;
            float m = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w][r]);
            const float ref = m == -INFINITY ? 0.f : m;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float lsum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(s_m[w][r] - ref);
                const float4 x = *reinterpret_cast<const float4 *>(smem + w * kOwn + (r * kPitch + d) * 4);
                lsum = fmaf(s_l[w][r], f, lsum);
                v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
            }
            if (all) {
                finish(r, d, v, m, lsum);
            } else {
                *reinterpret_cast<float4 *>(part + r * D + d) = v;
                if (d == 0) {
                    part[TR * D + r] = m;
                    part[TR * D + TR + r] = lsum;
                }
            }
        }
        if (!all) {
            // the last of the pair's CTAs to get here adds the parts, in their order
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int n = atomicAdd(p.counters + w0, 1);
                s_last = n == w1 - w0;
                if (s_last) p.counters[w0] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                add_parts<D, TR, kWarps * 32>(p, w0, w1, rows, r0, sh.row0, h);
            }
        }
        fence_async_smem();                                    // the ring was written to by threads; copies land in it next
        __syncthreads();
    }
    if (s_err) {                                               // a wait gave up: copies in flight land before the shared memory goes away
        for (int i = 0; i < 400; ++i) __nanosleep(256);
        if (tid == 0) atomicExch(p.status, s_err);
    }
}

// Dynamic shared memory of a CTA: rings, or the sums that take their place where those are longer.
static int smem_of(int NT, bool wide, int D) {
    const int sums = NT * 8 * (D + 4) * 4;
    return warps_of(NT, wide) * (sums > kRing ? sums : kRing);
}
static int grid_of(int NT, bool wide) {
    const int n = (wide ? 1 : (NT > 2 ? 2 : 3)) * jq_sm_count();
    return n < kJqCounters ? n : kJqCounters;
}
// Tiles of 8 query rows, by the rows that a key head has in a call.
static int tiles_of_rows(long long rows) { return rows <= 8 ? 1 : (rows <= 16 ? 2 : (rows <= 24 ? 3 : 4)); }
// Few pairs (sequence, key head) are cut into many parts, one for a CTA, and added by the last of them: CTAs of all an SM's warps leave a third
// as many parts.  us, wide / narrow, 64 query and 8 key heads of 128: 131071 tokens 61 / 70, eight sequences of 16000 54 / 61, four
// new tokens behind 16000 48 / 70.  With about as many pairs as SMs narrow CTAs hide one another's begin and end: 16 sequences of up to
// 4000 tokens, 3 to 5 new, 8 key heads of 64: 51 / 36.
static bool wide_of(long long pairs) { return 2 * pairs <= jq_sm_count(); }
// Query rows of a key head up to which attend_kernel is used, the kernel for prompts from there on.  us, attend_kernel / prompt_kernel, 64
// query and 8 key heads:
//     rows                              16         24         32         40         64
//     16 sequences of 2000, D = 128     45 / 54    43 / 55    70 / 53    90 / 54    91 / 54
//     1 of 16384, D = 128               30 / 44               49 / 48               70 / 48
//     64 of 1000, D = 64                39 / 91               50 / 89    91 / 92    94 / 91
static long long few_rows(int D) { return D == 64 ? 32 : 24; }
// Units that a CTA takes at least, about a stage for each warp: one row of 517 tokens, 32 heads: 9.7 us, 10.2 with two units, 16 with twelve.
constexpr int kLeast = 6;

typedef void (*attend_fn)(const AttendArgs);
template <int D, bool E4M3, int NT>
static attend_fn pick(bool wide) { return wide ? attend_kernel<D, E4M3, NT, true> : attend_kernel<D, E4M3, NT, false>; }
template <int D, bool E4M3>
static attend_fn pick(int NT, bool wide) {
    if (NT == 4) return pick<64, E4M3, 4>(wide);           // (no more than 24 rows at D = 128, see few_rows)
    return NT == 1 ? pick<D, E4M3, 1>(wide) : (NT == 2 ? pick<D, E4M3, 2>(wide) : pick<D, E4M3, 3>(wide));
}
template <int D>
static attend_fn pick(bool e4m3, int NT, bool wide) { return e4m3 ? pick<D, true>(NT, wide) : pick<D, false>(NT, wide); }

int check_cache(const jq_kv_cache *c, const jq_kv_batch *s);
Batch batch_of(const jq_kv_cache *c, const jq_kv_batch *s);
int most_new(const jq_kv_batch *s);

}  // namespace jqkv

using namespace jqkv;

extern "C" size_t jq_kv_attend_workspace_bytes(const jq_kv_cache *c, const jq_kv_batch *s, int q_heads) {
    if (check_cache(c, s) || q_heads <= 0) return 0;
    const long long rows = (long long)most_new(s) * (q_heads / c->kv_heads);
    if (rows > few_rows(c->head_dim)) return kJqData + prompt_workspace(c->head_dim);
    const int NT = tiles_of_rows(rows);
    return kJqData + 2 * (size_t)grid_of(NT, false) * NT * 8 * (c->head_dim + 2) * 4;        // (enough for wide CTAs, of which there are fewer)
}

extern "C" int jq_kv_attend(const jq_kv_cache *c, const jq_kv_batch *s, const void *q, const int64_t *stride_q, int q_heads,
                            float scale, int window, void *out, float *lse_or_null, int dtype, void *workspace,
                            size_t workspace_bytes, jq_stream_t stream) {
    return jq_kv_attend_status(c, s, q, stride_q, q_heads, scale, window, out, lse_or_null, dtype, workspace, workspace_bytes, nullptr, stream);
}

extern "C" int jq_kv_attend_status(const jq_kv_cache *c, const jq_kv_batch *s, const void *q, const int64_t *stride_q, int q_heads,
                                   float scale, int window, void *out, float *lse_or_null, int dtype, void *workspace,
                                   size_t workspace_bytes, int *status_or_null, jq_stream_t stream) {
    const int bad = check_cache(c, s);
    if (bad) return bad;
    if (dtype != JQ_F16 && dtype != JQ_BF16) return JQ_ERR_BAD_DTYPE;
    if (q_heads <= 0 || q_heads % c->kv_heads || window < 0 || !(scale > 0.f) || !(scale * kLog2e <= 3.4e38f)) return JQ_ERR_BAD_SHAPE;
    if (c->head_dim != 64 && c->head_dim != 128) return JQ_ERR_UNSUPPORTED;
    if (s->sequences == 0 || s->tokens == 0) return JQ_OK;
    if ((long long)most_new(s) * (q_heads / c->kv_heads) > (1 << 30)) return JQ_ERR_BAD_SHAPE;
    if (!q || !out || !stride_q || !workspace) return JQ_ERR_NULL_PTR;
    if ((reinterpret_cast<uintptr_t>(q) & 1u) || !jq_aligned16(out) || (reinterpret_cast<uintptr_t>(lse_or_null) & 3u) ||
        (reinterpret_cast<uintptr_t>(workspace) & 127u) || (reinterpret_cast<uintptr_t>(status_or_null) & 3u))
        return JQ_ERR_BAD_ALIGN;
    if (workspace_bytes < jq_kv_attend_workspace_bytes(c, s, q_heads)) return JQ_ERR_WORKSPACE;
    AttendArgs a{};
    a.b = batch_of(c, s);
    a.q = q; a.out = out; a.lse = lse_or_null;
    a.st = stride_q[0]; a.sh = stride_q[1];
    a.keys = reinterpret_cast<const uint8_t *>(c->keys); a.values = reinterpret_cast<const uint8_t *>(c->values);
    a.ks = c->key_scales; a.vs = c->value_scales;
    a.H = c->kv_heads; a.G = q_heads / c->kv_heads;
    a.window = (long long)window >= (long long)s->table_width * c->block_size ? 0 : window;      // (no sequence is longer)
    a.dtype = dtype;
    a.scale = scale * kLog2e;
    unsigned char *ws = reinterpret_cast<unsigned char *>(workspace);
    a.status = status_or_null ? status_or_null : reinterpret_cast<int *>(ws);
    a.counters = reinterpret_cast<int *>(ws + kJqHeader);
    a.parts = reinterpret_cast<float *>(ws + kJqData);
    const long long rows = (long long)most_new(s) * a.G;
    const bool e4m3 = c->fmt == JQ_KV_E4M3;
    if (rows > few_rows(c->head_dim)) {
        a.least = 8;
        return prompt_launch(a, c->head_dim, e4m3, reinterpret_cast<cudaStream_t>(stream));
    }
    const int NT = tiles_of_rows(rows);
    const bool wide = wide_of((long long)s->sequences * c->kv_heads);
    const int smem = smem_of(NT, wide, c->head_dim);
    const attend_fn kern = c->head_dim == 64 ? pick<64>(e4m3, NT, wide) : pick<128>(e4m3, NT, wide);
    static jq_contexts done[2][2][4][2];
    JQ_CUDA_TRY(jq_allow_smem(reinterpret_cast<const void *>(kern), smem, done[c->head_dim == 128][e4m3][NT - 1][wide]));
    a.least = kLeast;
    kern<<<grid_of(NT, wide), warps_of(NT, wide) * 32, smem, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    return jq_launch_status();
}
