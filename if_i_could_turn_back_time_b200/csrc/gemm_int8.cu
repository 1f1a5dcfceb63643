// Product of 8-bit integers with scales for each token and channel (sm_100a):
//   y[t][n] = (float(sum_k x[t][k] w[n][k]) * cs[n]) * ts[t] + bias[n],
// the sum exact in 32 bits (K up to 131071: |x w| <= 2^14), then three fp32 operations and the rounding to y's type.  As the
// integer sums are exact, no split of K and no order changes a bit of the result.
#include "rows8.cuh"

namespace jq8 {

using namespace jqta;

constexpr int kTileN = 128;            // weight rows of a tile: lanes of tensor memory
constexpr int kStep = 128;             // K of a stage: one 128-byte swizzle row of both operands
constexpr int kThreads = 192;          // 4 warps of outputs, a loader, an issuer of matrix instructions

struct GemmArgs {
    const float *cs, *ts, *bias;
    void *y;
    int *status;
    int N, T, steps, split, y_dtype, vec, early;
    int tiles_t, tiles_n, band;        // of a pair of CTAs
    int piece;                         // bytes that rows of y are multiples of: 16, 8, 4 or 2
};

// K-major operand tile in shared memory, 128-byte swizzle: atoms of 8 rows x 128 bytes, 1024 bytes apart
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)1 << 16 | (uint64_t)64 << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::i8 instruction descriptor: D = 32-bit integers, A = B = signed 8-bit, both K-major
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_i8_ss(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0;\n"
                 "  @q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
__device__ __forceinline__ int4 ld_cluster_i4(uint32_t addr, uint32_t rank) {
    int4 v;
    asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %4, %5; ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [a]; }"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// A sum with its scales and bias.  The channel's scale comes first: a packed one is 2^-107 at least, so that no product falls below fp32's normal
// numbers before the result does.
__device__ __forceinline__ float scaled(int sum, float cs, float ts, float bias) { return fmaf(__int2float_rn(sum) * cs, ts, bias); }
// Where a channel's scale is above 2^64, so that the product could leave the range on the other side, it is held 2^-64 times as large and has one
// rounding more.  (By a test of every scale in one function: 10000 x 300 x 2500 35 us instead of 30.)
constexpr float kLarge = 18446744073709551616.f, kLargeInverse = 5.421010862427522e-20f;
__device__ __forceinline__ float scaled_large(int sum, float cs, float ts, float bias) {
    return fabsf(cs) > kLarge ? fmaf(__int2float_rn(sum) * (cs * kLargeInverse) * ts, kLarge, bias) : scaled(sum, cs, ts, bias);
}

template <class T>
__device__ __forceinline__ void store4(T *y, const float (&v)[4], int n, bool vec) {
    if (vec && n >= 4) {
        alignas(16) const T r[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(r);
        else *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(r);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (k < n) y[k] = (T)v[k];
}

template <int NT> struct Few {
    static constexpr int kStage = (kTileN + NT) * kStep;
    static constexpr int kStages = NT == 128 ? 3 : (NT == 64 ? 4 : (NT == 32 ? 5 : 6));
    static constexpr int kRing = kStage * kStages;
    static constexpr int kSmem = kRing + 1024 + 256;
    static constexpr int kCols = NT < 32 ? 32 : NT;
    static_assert(kRing >= NT * kTileN * 4, "the tile's sums pass through the ring");
};

// Few tokens: tiles of 128 channels x NT tokens, the weights as the operand of 128 rows, so that what a stage costs in shared memory and time
// goes by the tokens that there are.  Bound by reading the weights: two CTAs an SM with some 100 KB of copies in flight each.  Where there are few
// tiles the CTAs of a cluster share a tile's K range, and their sums meet in distributed shared memory (whole numbers: any split gives the
// same bits).  28672 x 8192, 48 tokens: 43 us, 5.5 TB/s; 11008 x 4096, one token: 10.2 us in three parts (11.4 in one, 12.2 in two: 172 CTAs load
// some SMs twice), of which the launch, set-up and exchange are some 3.
template <int NT>
__global__ void __launch_bounds__(kThreads) gemm_int8_kernel(const __grid_constant__ GemmArgs p, const __grid_constant__ CUtensorMap wmap,
                                                             const __grid_constant__ CUtensorMap xmap) {
    using C = Few<NT>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_err;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, bars = ring + C::kRing;
    auto full = [&](int s) { return bars + 8u * s; };
    auto free_ = [&](int s) { return bars + 8u * (C::kStages + s); };
    const uint32_t done = bars + 8u * (2 * C::kStages);
    volatile int *err = &s_err;
    if (tid == 0) {
        s_err = 0;
        for (int s = 0; s < C::kStages; ++s) { mbar_init(full(s), 1); mbar_init(free_(s), 1); }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(C::kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const int rank = p.split > 1 ? (int)(blockIdx.x % p.split) : 0;
    const int n0 = blockIdx.x / p.split * kTileN, t0 = blockIdx.y * NT;
    const int k_lo = p.steps * rank / p.split, count = p.steps * (rank + 1) / p.split - k_lo;
    pdl_launch_dependents();

    if (warp == 4) {
        if (lane == 0) {
            auto load_w = [&](int i, int s) {
                mbar_expect_tx(full(s), C::kStage);
                tma_2d_g2s(ring + s * C::kStage, &wmap, (k_lo + i) * kStep, n0, full(s));
            };
            auto load_x = [&](int i, int s) {
                tma_2d_g2s(ring + s * C::kStage + kTileN * kStep, &xmap, (k_lo + i) * kStep, t0, full(s));
            };
            // Weights that no kernel of this call writes are asked for while the activation is still being quantised
            const int ahead = min(C::kStages, count);
            if (!p.early) pdl_wait();
            for (int i = 0; i < ahead; ++i) load_w(i, i);
            if (p.early) pdl_wait();
            for (int i = 0; i < ahead; ++i) load_x(i, i);
            int s = 0;
            uint32_t par = 0;
            for (int i = ahead; i < count; ++i) {
                if (!mbar_wait(free_(s), par, err)) break;
                load_w(i, s);
                load_x(i, s);
                if (++s == C::kStages) { s = 0; par ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        const uint32_t elected = elect_one();
        constexpr uint32_t idesc = idesc_i8(kTileN, NT);
        pdl_wait();                                        // (the bounded waits do not count the kernel in front of this one)
        int s = 0;
        uint32_t par = 0;
        bool ok = true;
        for (int i = 0; i < count; ++i) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(full(s), par, err)))) break;
            tc_fence_after();
            const uint64_t a = desc_sw128(ring + s * C::kStage), b = desc_sw128(ring + s * C::kStage + kTileN * kStep);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_i8_ss(elected, tmem, a + 2 * k, b + 2 * k, idesc, i > 0 || k > 0);
            mma_commit(elected, free_(s));
            if (++s == C::kStages) { s = 0; par ^= 1; }
        }
        if (ok) mma_commit(elected, done);
    } else {
        // sums -> shared memory, [token][channel]: every stage has been read once the last instruction is done
        pdl_wait();
        if (__all_sync(0xffffffffu, mbar_wait(done, 0, err))) {
            tc_fence_after();
            const uint32_t to = ring + (warp * 32 + lane) * 4;
#pragma unroll 1
            for (int c = 0; c < NT; c += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + (c + k) * (kTileN * 4)), "r"(r[k]) : "memory");
            }
        }
        __syncwarp();
    }
    pdl_wait();
    if (p.split > 1) cluster_sync();
    else __syncthreads();
    if (!*err) {
        const int n = n0 + lane * 4, left = p.N - n;
        const int lo = NT * rank / p.split, hi = min(NT * (rank + 1) / p.split, p.T - t0);
        float cs[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cs[k] = k < left ? p.cs[n + k] : 0.f;
            b[k] = k < left && p.bias ? p.bias[n + k] : 0.f;
        }
        float ts = lo + warp < hi ? p.ts[t0 + lo + warp] : 0.f;         // (a token's scale is asked for while others are used)
        const bool large = fmaxf(fmaxf(fabsf(cs[0]), fabsf(cs[1])), fmaxf(fabsf(cs[2]), fabsf(cs[3]))) > kLarge;
        for (int t = lo + warp; t < hi; t += kThreads / 32) {
            const uint32_t from = ring + t * (kTileN * 4) + lane * 16;
            int4 a;
            if (p.split == 1) {
                const uint4 u = lds128(from);
                a = make_int4((int)u.x, (int)u.y, (int)u.z, (int)u.w);
            } else {
                a = make_int4(0, 0, 0, 0);
                for (int r = 0; r < p.split; ++r) {
                    const int4 u = ld_cluster_i4(from, (uint32_t)r);
                    a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
                }
            }
            float v[4] = {scaled(a.x, cs[0], ts, b[0]), scaled(a.y, cs[1], ts, b[1]), scaled(a.z, cs[2], ts, b[2]), scaled(a.w, cs[3], ts, b[3])};
            if (large) {
                v[0] = scaled_large(a.x, cs[0], ts, b[0]); v[1] = scaled_large(a.y, cs[1], ts, b[1]);
                v[2] = scaled_large(a.z, cs[2], ts, b[2]); v[3] = scaled_large(a.w, cs[3], ts, b[3]);
            }
            if (t + kThreads / 32 < hi) ts = p.ts[t0 + t + kThreads / 32];
            const size_t at = (size_t)(t0 + t) * p.N + n;
            if (p.y_dtype == JQ_F32) store4(reinterpret_cast<float *>(p.y) + at, v, left, p.vec);
            else if (p.y_dtype == JQ_F16) store4(reinterpret_cast<__half *>(p.y) + at, v, left, p.vec);
            else store4(reinterpret_cast<__nv_bfloat16 *>(p.y) + at, v, left, p.vec);
        }
    } else {   // a wait gave up: let the copies still in flight land before the CTA's shared memory goes away
        for (int i = 0; i < 400; ++i) __nanosleep(256);
        if (tid == 0) atomicExch(p.status, *err);
    }
    tc_fence_before();
    if (p.split > 1) cluster_sync();         // (the others may still be reading this CTA's sums)
    else __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols) : "memory");
    }
}

// ---- many tokens: a pair of CTAs per tile ------------------------------------------------

constexpr int kPairThreads = 320;      // 8 warps of outputs, a loader, an issuer
constexpr int kPitch = 80;             // bytes between a warp's rows of outputs in shared memory (64 of them, spread over the banks)

template <int BN> struct Pair {
    static constexpr int kStage = (128 + BN / 2) * kStep;          // of each CTA: 128 tokens, half of the channels
    static constexpr int kStages = BN == 256 ? 6 : 8;
    static constexpr int kRing = kStage * kStages;
    static constexpr int kOut = 8 * (32 * kPitch + BN * 4);        // a warp's outputs, and its BN / 2 columns' scales and biases
    static_assert(kRing >= BN * 128 * 4, "a tile's sums pass through the ring where CTAs share its K range");
    static constexpr int kSmem = kRing + kOut + 1024 + 256;
};

__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// A box into this CTA's shared memory, counted on a barrier of either CTA of the pair
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const void *tmap, int x, int y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0;\n"
                 "  @q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p; }"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
// What has been issued so far is done: told to the barrier at this place of both CTAs
__device__ __forceinline__ void commit_pair(uint32_t elected, uint32_t bar, uint32_t both) {
    asm volatile("{ .reg .pred q; setp.ne.b32 q, %1, 0;\n"
                 "  @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2; }"
                 ::"r"(bar), "r"(elected), "h"((uint16_t)both) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 64 bytes of 32 rows from a warp's shared memory into rows of y, in pieces of W bytes that rows of y are multiples of
template <int W>
__device__ __forceinline__ void store_rows(const GemmArgs &p, uint32_t out, int t0, int nb, int row_bytes, int lane) {
    constexpr int kLanes = 64 / W, kRows = 32 / kLanes;
    const int b = nb + lane % kLanes * W;
    const uint32_t from = out + lane / kLanes * kPitch + lane % kLanes * W;
    unsigned char *y = reinterpret_cast<unsigned char *>(p.y) + (size_t)(t0 + lane / kLanes) * row_bytes + b;
    const int left = p.T - t0 - lane / kLanes;
#pragma unroll 8
    for (int i = 0; i < 32; i += kRows) {
        const bool in = i < left && b < row_bytes;
        if constexpr (W == 16) {
            const uint4 u = lds128(from + i * kPitch);
            if (in) *reinterpret_cast<uint4 *>(y) = u;
        } else if constexpr (W == 8) {
            uint2 u;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(from + i * kPitch));
            if (in) *reinterpret_cast<uint2 *>(y) = u;
        } else if constexpr (W == 4) {
            const uint32_t u = lds32(from + i * kPitch);
            if (in) *reinterpret_cast<uint32_t *>(y) = u;
        } else {
            unsigned short u;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(from + i * kPitch));
            if (in) *reinterpret_cast<unsigned short *>(y) = u;
        }
        y += (size_t)kRows * row_bytes;
    }
}

// 32 columns of a warp's 32 tokens (a token per lane): scaled, turned in shared memory 64 bytes of a row at a time, and written as rows
template <class T>
__device__ __forceinline__ void write32(const GemmArgs &p, const uint32_t (&r)[32], uint32_t out, uint32_t scales, uint32_t biases, float ts, int t0, int n0, int lane) {
    constexpr int kCols = 64 / (int)sizeof(T);
#pragma unroll
    for (int half = 0; half < 32 / kCols; ++half) {
        float v[kCols];
#pragma unroll
        for (int c = 0; c < kCols; c += 4) {
            const uint4 cs = lds128(scales + (half * kCols + c) * 4);
            const uint32_t *s = &cs.x;
            uint4 b4 = make_uint4(0, 0, 0, 0);
            if (p.bias) b4 = lds128(biases + (half * kCols + c) * 4);
            const uint32_t *b = &b4.x;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[c + k] = scaled((int)r[half * kCols + c + k], __uint_as_float(s[k]), ts, __uint_as_float(b[k]));
        }
        __syncwarp();
        const uint32_t row = out + lane * kPitch;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t w[4];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = __float_as_uint(v[4 * q + k]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = pack2<T>(v[8 * q + 2 * k], v[8 * q + 2 * k + 1]);
            }
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + 16 * q), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        __syncwarp();
        const int nb = (n0 + half * kCols) * (int)sizeof(T), row_bytes = p.N * (int)sizeof(T);
        if (p.piece == 16) store_rows<16>(p, out, t0, nb, row_bytes, lane);
        else if (p.piece == 8) store_rows<8>(p, out, t0, nb, row_bytes, lane);
        else if (p.piece == 4) store_rows<4>(p, out, t0, nb, row_bytes, lane);
        else if constexpr (sizeof(T) == 2) store_rows<2>(p, out, t0, nb, row_bytes, lane);
    }
}

// The same of channels of which one has a scale above kLarge, by elements; t: the lane's token
__device__ __forceinline__ void write32_large(const GemmArgs &p, const uint32_t (&r)[32], uint32_t scales, uint32_t biases, float ts, int t, int n0) {
#pragma unroll
    for (int k = 0; k < 32; ++k)
        if (t < p.T && n0 + k < p.N)
            jq::store_out(p.y, (size_t)t * p.N + n0 + k, scaled_large((int)r[k], __uint_as_float(lds32(scales + 4 * k)), ts, __uint_as_float(lds32(biases + 4 * k))), p.y_dtype);
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// Tiles of 256 tokens x BN channels on a pair of CTAs (cta_group::2): each holds the sums of its 128 tokens, and both read one another's
// half of the weights, so that an SM's shared memory takes in half of the operand bytes per product.  Persistent; the sums of a tile are
// scaled and written while the next one is multiplied.  Where there are few tiles, the pairs of a cluster share a tile's K range
// instead (split > 1): their sums meet in distributed shared memory, a part of the columns in each.
// Bound by the tensor core: a stage of 128 values takes 520 to 560 clocks (512 are its products') with 256 channels, 400 to 450 (256) with 128,
// which ask the L2 for 24 KB in that time.  8192 x 8192 x 28672: 1100 us in a few calls (3.5 POP/s, 1.06 of twice the measured bf16 rate),
// 1270 in calls one behind another for seconds, when the power cap holds the clock down (3.0 POP/s, 0.92 of that rate, 1.11 of twice the bf16 rate
// measured the same way); 2048 x 4096 x 11008: 60 and 70 us, 344 tiles on 74 pairs being 4.65 waves.  (Single CTAs of 128 x 256: 2098 and 121.)
template <int BN>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm_int8_pair_kernel(const __grid_constant__ GemmArgs p, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
    using C = Pair<BN>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_err;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t rank = cta_rank() & 1, leader = cta_rank() & ~1u;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, outs = ring + C::kRing, bars = outs + C::kOut;
    auto full = [&](int s) { return bars + 8u * s; };                                  // (the leader's: both CTAs' boxes)
    auto free_ = [&](int s) { return bars + 8u * (C::kStages + s); };
    auto ready = [&](int a) { return bars + 8u * (2 * C::kStages + a); };              // sums complete
    auto taken = [&](int a) { return bars + 8u * (2 * C::kStages + 2 + a); };          // (the leader's) read by both CTAs' warps
    volatile int *err = &s_err;
    if (tid == 0) {
        s_err = 0;
        for (int s = 0; s < C::kStages; ++s) { mbar_init(full(s), 1); mbar_init(free_(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(ready(a), 1); mbar_init(taken(a), 16); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    pdl_launch_dependents();

    const int width = 2 * p.split, clusters = gridDim.x / width, first = blockIdx.x / width;     // (split > 1: a tile per cluster)
    const int tiles = p.tiles_t * p.tiles_n;
    const int part = (int)(leader >> 1);                   // of the K range
    const int k_lo = p.steps * part / p.split, steps = p.steps * (part + 1) / p.split - k_lo;
    // tiles in groups of `band` rows of tokens, which stay in the L2 while the weights pass by
    auto place = [&](int tile, int &t0, int &n0) {
        const int per = p.band * p.tiles_n, g = tile / per, in = tile - g * per;
        const int rows = min(p.band, p.tiles_t - g * p.band);
        t0 = (g * p.band + in % rows) * 256 + (int)rank * 128;
        n0 = in / rows * BN;
    };
    const int quarter = warp & 3, side = warp >> 2;        // of an output warp: lanes of tensor memory, half of the columns
    const uint32_t out = outs + warp * (32 * kPitch + BN * 4), scales = out + 32 * kPitch, biases = scales + BN * 2;
    // scales and biases of `cols` columns from n on into the warp's shared memory; whether a scale is above kLarge
    auto take_params = [&](int n, int cols) -> bool {
        float most = 0.f;
        __syncwarp();
        for (int c = lane; c < cols; c += 32) {
            const float cs = n + c < p.N ? p.cs[n + c] : 0.f, b = n + c < p.N && p.bias ? p.bias[n + c] : 0.f;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + c * 4), "f"(cs) : "memory");
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(biases + c * 4), "f"(b) : "memory");
            most = fmaxf(most, fabsf(cs));
        }
        __syncwarp();
        return __any_sync(0xffffffffu, most > kLarge);
    };
    auto write = [&](const uint32_t (&r)[32], int c, float ts, int t0, int n0) {      // c: among the warp's columns
        if (t0 >= p.T || n0 + c >= p.N) return;
        if (p.y_dtype == JQ_F32) write32<float>(p, r, out, scales + c * 4, biases + c * 4, ts, t0, n0 + c, lane);
        else if (p.y_dtype == JQ_F16) write32<__half>(p, r, out, scales + c * 4, biases + c * 4, ts, t0, n0 + c, lane);
        else write32<__nv_bfloat16>(p, r, out, scales + c * 4, biases + c * 4, ts, t0, n0 + c, lane);
    };

    if (warp == 8) {
        if (lane == 0) {
            const uint32_t stage_bytes = 2 * C::kStage;
            int s = 0, ahead = 0;
            uint32_t par = 1;                              // (the first round finds every stage free)
            bool ok = true;
            auto load_w = [&](int n0, int i, int s_) {
                if (rank == 0) mbar_expect_tx(full(s_), stage_bytes);
                tma_2d_pair(ring + s_ * C::kStage + 128 * kStep, &wmap, (k_lo + i) * kStep, n0 + (int)rank * (BN / 2), at_rank(full(s_), leader));
            };
            // Weights that no kernel of this call writes are asked for while the activation is still being quantised
            if (p.early && first < tiles) {
                int t0, n0;
                place(first, t0, n0);
                ahead = min(C::kStages, steps);
                for (int i = 0; i < ahead; ++i) load_w(n0, i, i);
            }
            pdl_wait();
            for (int tile = first; tile < tiles && ok; tile += clusters) {
                int t0, n0;
                place(tile, t0, n0);
                for (int i = 0; i < steps; ++i) {
                    if (ahead > 0) --ahead;
                    else {
                        if (!(ok = mbar_wait(free_(s), par, err))) break;
                        load_w(n0, i, s);
                    }
                    tma_2d_pair(ring + s * C::kStage, &xmap, (k_lo + i) * kStep, t0, at_rank(full(s), leader));
                    if (++s == C::kStages) { s = 0; par ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        if (rank == 0) {
            const uint32_t elected = elect_one();
            constexpr uint32_t idesc = idesc_i8(256, BN);
            const uint32_t both = 3u << leader;
            pdl_wait();                                    // (the bounded waits do not count the kernel in front of this one)
            auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, err)); };
            int s = 0, a = 0;
            uint32_t par = 0, a_par = 1;                   // (the first wait on free sums passes at once)
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += clusters) {
                if (!(ok = wait(taken(a), a_par))) break;
                tc_fence_after();
                const uint32_t d = tmem + a * BN;
                for (int i = 0; i < steps; ++i) {
                    if (!(ok = wait(full(s), par))) break;
                    tc_fence_after();
                    const uint64_t da = desc_sw128(ring + s * C::kStage), db = desc_sw128(ring + s * C::kStage + 128 * kStep);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_i8_pair(elected, d, da + 2 * k, db + 2 * k, idesc, i > 0 || k > 0);
                    commit_pair(elected, free_(s), both);
                    if (++s == C::kStages) { s = 0; par ^= 1; }
                }
                if (!ok) break;
                commit_pair(elected, ready(a), both);
                if (++a == 2) { a = 0; a_par ^= 1; }
            }
        }
    } else if (p.split == 1) {
        pdl_wait();
        int a = 0;
        uint32_t par = 0;
        for (int tile = first; tile < tiles; tile += clusters) {
            int t0, n0;
            place(tile, t0, n0);
            t0 += quarter * 32;
            n0 += side * (BN / 2);
            const float ts = t0 + lane < p.T ? p.ts[t0 + lane] : 0.f;
            const bool large = take_params(n0, BN / 2);
            if (!__all_sync(0xffffffffu, mbar_wait(ready(a), par, err))) break;
            tc_fence_after();
            const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + a * BN + side * (BN / 2);
            if (large) {
#pragma unroll 1
                for (int j = 0; j < BN / 64; ++j) {
                    uint32_t r[32];
                    tmem_ld32(from + j * 32, r);
                    tmem_wait_ld();
                    write32_large(p, r, scales + j * 128, biases + j * 128, ts, t0 + lane, n0 + j * 32);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_cluster(at_rank(taken(a), leader));
                if (++a == 2) { a = 0; par ^= 1; }
                continue;
            }
            uint32_t r[2][32];
            tmem_ld32(from, r[0]);
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) {
                tmem_wait_ld();
                if (j + 1 < BN / 64) tmem_ld32(from + (j + 1) * 32, r[(j + 1) & 1]);
                else {                                     // all of this warp's sums are in registers
                    tc_fence_before();
                    if (lane == 0) arrive_cluster(at_rank(taken(a), leader));
                }
                write(r[j & 1], j * 32, ts, t0, n0);
            }
            if (++a == 2) { a = 0; par ^= 1; }
        }
    } else {
        // sums -> shared memory, [column][token]: every stage has been read once the last instruction is done
        pdl_wait();
        if (__all_sync(0xffffffffu, mbar_wait(ready(0), 0, err))) {
            tc_fence_after();
            const uint32_t to = ring + (quarter * 32 + lane) * 4;
#pragma unroll 1
            for (int c = side * (BN / 2); c < (side + 1) * (BN / 2); c += 32) {
                uint32_t r[32];
                tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + (c + k) * 512), "r"(r[k]) : "memory");
            }
        }
    }
    __syncwarp();
    if (p.split > 1) {
        cluster_sync();
        if (warp < 8 && !*err) {
            const int cols = BN / p.split / 2, c_lo = part * (BN / p.split) + side * cols;      // of this warp
            int t0, n0;
            place(first, t0, n0);
            t0 += quarter * 32;
            n0 += c_lo;
            const float ts = t0 + lane < p.T ? p.ts[t0 + lane] : 0.f;
            const bool large = take_params(n0, cols);
            for (int c = 0; c < cols; c += 32) {
                uint32_t r[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) r[k] = 0;
#pragma unroll 1
                for (int o = 0; o < p.split; ++o) {
                    const uint32_t from = at_rank(ring + (quarter * 32 + lane) * 4, 2 * (uint32_t)o + rank) + (uint32_t)(c_lo + c) * 512;
#pragma unroll
                    for (int k = 0; k < 32; ++k) r[k] += ld_cluster_u32(from + k * 512);
                }
                if (large) write32_large(p, r, scales + c * 4, biases + c * 4, ts, t0 + lane, n0 + c);
                else write(r, c, ts, t0, n0);
            }
        }
        __syncwarp();
    }
    if (*err) {   // a wait gave up: let the copies and products still in flight end before the pair's shared memory goes away
        for (int i = 0; i < 400; ++i) __nanosleep(256);
        if (lane == 0) atomicExch(p.status, *err);
    }
    tc_fence_before();
    cluster_sync();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
    }
}

// ---- host side -------------------------------------------------------------------------

static int encode(CUtensorMap *map, const void *base, int rows, int K, int64_t stride, int box_rows) {
    ta_encode_fn enc = ta_encoder();
    if (!enc) return JQ_ERR_UNSUPPORTED;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)kStep, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? JQ_OK : JQ_ERR_CUDA_BASE - (int)cudaErrorInvalidValue;
}

struct Form { bool pair; int tile, split; };   // tile: tokens of a single CTA's tile, channels of a pair's

// Which kernel, tile and split of K, by a model of the time in us: what a launch, a tile's outputs, a stage of 128 values of K and an exchange
// between CTAs take.  Its constants are fitted to 2524 timed calls (18 numbers of tokens up to 10000, 14 matrices from 100 x 300 to
// 32000 x 2048 and 28672 x 8192, every form): the choice is 1.0 % behind the best form on average, 15 % at most.  Both sides of its turns, us:
//   4096 x 4096         T = 64    single CTAs of 64 tokens, K in four parts 9.6     pairs of 128 channels, two parts 10.5, one 10.9
//                       T = 256   single 14.0 (128 tokens, four parts)              pairs of 128 channels, two parts 11.0, one 11.5
//                       T = 1024  single 20.1                                       pairs of 128 18.7, of 256 16.5
//   28672 x 8192        T = 64    single 44                                         pairs of 256 53
//                       T = 200   single 84                                         pairs of 256 57
//   100 x 300           T = 512   single, 32 tokens 4.1                             pairs of 128 5.4
static Form choose_form(int N, int K, int T, int steps, int sms) {
    Form best{false, 16, 1};
    double least = 0;
    auto offer = [&](bool pair, int tile, int split, double us) {
        if (least == 0 || us < least) { best = Form{pair, tile, split}; least = us; }
    };
    for (int nt = 16; nt <= 128; nt *= 2) {
        // (tiles of 32 tokens for more than 32 only where the weights are next to nothing: 300 x 784, T = 200, 4.7 and in tiles of 64 5.1; between that
        // and the bound nothing was timed)
        if ((T <= nt / 2 && nt > 16) || (T > nt && (nt < 32 || (nt == 32 && (long long)N * K >= 600000)))) continue;
        const long long tiles = (long long)((N + kTileN - 1) / kTileN) * ((T + nt - 1) / nt);
        for (int s = 1; s <= 8; s = s == 4 ? 8 : s + 1) {
            const long long ctas = tiles * s, room = s == 8 ? sms / 18 * 32 : 2 * sms;      // (clusters of eight: two in the 16 or 18 SMs of a GPC, twice)
            if (s > steps || (ctas > room && (s > 1 || T > 64))) break;
            const double turns = (double)(ctas / room * 2 + (ctas % room + sms - 1) / sms);       // CTAs that an SM has, one behind another
            offer(false, nt, s, 2.16 + 0.030 * nt + turns * ((steps + s - 1) / s) * (0.2045 + 0.0008 * nt) + (s > 1 ? 0.034 * nt : 0.0));
        }
    }
    if (T > 64)
        for (int bn = 256; bn >= 128; bn /= 2) {
            const long long tiles = (long long)((N + bn - 1) / bn) * ((T + 255) / 256);
            for (int s = 1; s <= bn / 64; s *= 2) {                                            // (32 columns for each of a CTA's output warps at least)
                const long long room = s == 1 ? sms / 2 : sms / 18 * (s == 2 ? 4 : 2);
                if (s > steps || (s > 1 && tiles > room)) break;
                const double waves = (double)((tiles + room - 1) / room);
                offer(true, bn, s, 2.78 + bn / 128 * (0.22 + 1.25 * waves + (s > 1 ? 2.68 : 0.0)) + waves * ((steps + s - 1) / s) * (bn == 256 ? 0.294 : 0.207));
            }
        }
    return best;
}

template <int NT>
static int launch(GemmArgs &a, const void *w, int64_t w_stride, const void *x, int64_t x_stride, int K, cudaStream_t st) {
    CUtensorMap wmap, xmap;
    int rc = encode(&wmap, w, a.N, K, w_stride, kTileN);
    if (!rc) rc = encode(&xmap, x, a.T, K, x_stride, NT);
    if (rc) return rc;
    const int tiles = (a.N + kTileN - 1) / kTileN, across = (a.T + NT - 1) / NT;
    static jq_contexts done;
    auto kern = gemm_int8_kernel<NT>;
    JQ_CUDA_TRY(jq_allow_smem(reinterpret_cast<const void *>(kern), Few<NT>::kSmem, done));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * a.split), (unsigned)across);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Few<NT>::kSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = a.split > 1 ? 2 : 1;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, wmap, xmap));
    return jq_launch_status();
}

template <int BN>
static int launch_pair(GemmArgs &a, const void *w, int64_t w_stride, const void *x, int64_t x_stride, int K, cudaStream_t st) {
    CUtensorMap wmap, xmap;
    int rc = encode(&wmap, w, a.N, K, w_stride, BN / 2);
    if (!rc) rc = encode(&xmap, x, a.T, K, x_stride, 128);
    if (rc) return rc;
    a.tiles_t = (a.T + 255) / 256;
    a.tiles_n = (a.N + BN - 1) / BN;
    a.band = 16;
    const uintptr_t rows = reinterpret_cast<uintptr_t>(a.y) | (uintptr_t)a.N * (a.y_dtype == JQ_F32 ? 4 : 2);
    a.piece = rows % 16 == 0 ? 16 : rows % 8 == 0 ? 8 : rows % 4 == 0 ? 4 : 2;
    static jq_contexts done;
    auto kern = gemm_int8_pair_kernel<BN>;
    JQ_CUDA_TRY(jq_allow_smem(reinterpret_cast<const void *>(kern), Pair<BN>::kSmem, done));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2 * (unsigned)a.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    const long long tiles = (long long)a.tiles_t * a.tiles_n;
    const int pairs = jq_sm_count() / 2;
    cfg.gridDim = dim3(2 * (unsigned)(a.split > 1 ? tiles * a.split : (tiles < pairs ? tiles : pairs)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = Pair<BN>::kSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, wmap, xmap));
    return jq_launch_status();
}

// early: the kernel in front of this one on the stream is one of this call, so that the weights are settled
static int multiply(const void *w, const float *cs, const void *x, int64_t x_stride, const float *ts, const float *bias, void *y, int N, int K,
                    int T, int y_dtype, int *status, bool early, cudaStream_t st) {
    GemmArgs a{};
    a.cs = cs; a.ts = ts; a.bias = bias; a.y = y; a.status = status; a.N = N; a.T = T; a.steps = (K + kStep - 1) / kStep;
    a.y_dtype = y_dtype; a.early = early;
    a.vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & (y_dtype == JQ_F32 ? 15u : 7u)) == 0;
    const int64_t ws = jq_row_stride_codes(K);
    const Form f = choose_form(N, K, T, a.steps, jq_sm_count());
    a.split = f.split;
    if (f.pair) return f.tile == 256 ? launch_pair<256>(a, w, ws, x, x_stride, K, st) : launch_pair<128>(a, w, ws, x, x_stride, K, st);
    if (f.tile == 16) return launch<16>(a, w, ws, x, x_stride, K, st);
    if (f.tile == 32) return launch<32>(a, w, ws, x, x_stride, K, st);
    if (f.tile == 64) return launch<64>(a, w, ws, x, x_stride, K, st);
    return launch<128>(a, w, ws, x, x_stride, K, st);
}

static int check(const void *w, const float *cs, const float *bias, const void *y, const int *status, int N, int K, int B, int y_dtype) {
    if (!w || !cs || !y || !status) return JQ_ERR_NULL_PTR;
    if (N <= 0 || K <= 0 || B <= 0 || B > JQ_INT8_MAX_ROWS || K > JQ_INT8_MAX_K || N > (1 << 28)) return JQ_ERR_BAD_SHAPE;
    if (y_dtype < 0 || y_dtype > 2) return JQ_ERR_BAD_DTYPE;
    return jq_aligned16(w) && jq_whole(cs, 4) && jq_whole(bias, 4) && jq_whole(y, y_dtype == JQ_F32 ? 4 : 2) && jq_whole(status, 4) ? JQ_OK : JQ_ERR_BAD_ALIGN;
}

static size_t scale_room(int rows) { return ((size_t)rows * 4 + 255) / 256 * 256; }

}  // namespace jq8

using namespace jq8;

extern "C" size_t jq_int8_scratch_bytes(int B, int K) {
    if (B <= 0 || K <= 0 || K > JQ_INT8_MAX_K) return 0;
    return scale_room(B) + (size_t)B * jq_row_stride_codes(K);
}

extern "C" int jq_int8_form(int N, int K, int B, int *pair, int *tile, int *split) {
    if (!pair || !tile || !split) return JQ_ERR_NULL_PTR;
    if (N <= 0 || K <= 0 || B <= 0 || B > JQ_INT8_MAX_ROWS || K > JQ_INT8_MAX_K || N > (1 << 28)) return JQ_ERR_BAD_SHAPE;
    const Form f = choose_form(N, K, B, (K + kStep - 1) / kStep, jq_sm_count());
    *pair = f.pair; *tile = f.tile; *split = f.split;
    return JQ_OK;
}

extern "C" int jq_int8_linear(const void *qweight, const float *scales, const void *x, const float *bias, void *y, int N, int K, int B,
                              int had_block, int x_dtype, int y_dtype, void *scratch, size_t scratch_size, int *status, jq_stream_t stream) {
    if (!x || !scratch) return JQ_ERR_NULL_PTR;
    int rc = check(qweight, scales, bias, y, status, N, K, B, y_dtype);
    if (rc) return rc;
    if (scratch_size < jq_int8_scratch_bytes(B, K)) return JQ_ERR_WORKSPACE;
    if (!jq_aligned16(scratch)) return JQ_ERR_BAD_ALIGN;
    float *ts = reinterpret_cast<float *>(scratch);
    void *codes = reinterpret_cast<unsigned char *>(scratch) + scale_room(B);
    rc = jq_quantize_rows(x, K, B, K, had_block, x_dtype, codes, jq_row_stride_codes(K), ts, stream);
    if (rc) return rc;
    return multiply(qweight, scales, codes, jq_row_stride_codes(K), ts, bias, y, N, K, B, y_dtype, status, true, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int jq_int8_matmul(const void *qweight, const float *scales, const void *codes, int64_t code_stride, const float *row_scales,
                              const float *bias, void *y, int N, int K, int B, int y_dtype, int *status, jq_stream_t stream) {
    if (!codes || !row_scales) return JQ_ERR_NULL_PTR;
    const int rc = check(qweight, scales, bias, y, status, N, K, B, y_dtype);
    if (rc) return rc;
    if (code_stride < K) return JQ_ERR_BAD_SHAPE;
    if (!jq_aligned16(codes) || code_stride % 16 || !jq_whole(row_scales, 4)) return JQ_ERR_BAD_ALIGN;
    return multiply(qweight, scales, codes, code_stride, row_scales, bias, y, N, K, B, y_dtype, status, false, reinterpret_cast<cudaStream_t>(stream));
}
