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

template <class T>
__device__ __forceinline__ void store4(T *y, const float (&v)[4], int n, bool vec) {
    if (vec && n >= 4) {
        T r[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
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
    static constexpr int kStages = NT == 256 ? 4 : (NT == 128 ? 3 : (NT == 64 ? 4 : (NT == 32 ? 5 : 6)));
    static constexpr int kRing = kStage * kStages;
    static constexpr int kSmem = kRing + 1024 + 256;
    static constexpr int kCols = NT < 32 ? 32 : NT;
    static_assert(kRing >= NT * kTileN * 4, "the tile's sums pass through the ring");
};

// Tiles of 128 channels x NT tokens, the weights as the operand of 128 rows: what a stage costs in shared memory and time goes by the
// tokens that there are.  The CTAs of a cluster share a tile's K range; their sums meet in distributed shared memory.
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
            // (the channel's scale first: weights are of a moderate size, so that neither product leaves fp32's range before the result does)
            const float ts = p.ts[t0 + t];
            const float v[4] = {fmaf(__int2float_rn(a.x) * cs[0], ts, b[0]), fmaf(__int2float_rn(a.y) * cs[1], ts, b[1]),
                                fmaf(__int2float_rn(a.z) * cs[2], ts, b[2]), fmaf(__int2float_rn(a.w) * cs[3], ts, b[3])};
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

// CTAs that share a tile's K range: as many as give every SM about two CTAs with at least two stages each
static int split_of(long long tiles, int steps, int sms) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= 2 * sms && steps >= 4 * s) s *= 2;
    return s;
}

template <int NT>
static int launch(GemmArgs &a, const void *w, int64_t w_stride, const void *x, int64_t x_stride, int K, cudaStream_t st) {
    CUtensorMap wmap, xmap;
    int rc = encode(&wmap, w, a.N, K, w_stride, kTileN);
    if (!rc) rc = encode(&xmap, x, a.T, K, x_stride, NT);
    if (rc) return rc;
    const int tiles = (a.N + kTileN - 1) / kTileN, across = (a.T + NT - 1) / NT;
    a.split = split_of((long long)tiles * across, a.steps, jq_sm_count());
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

// early: the kernel in front of this one on the stream is one of this call, so that the weights are settled
static int multiply(const void *w, const float *cs, const void *x, int64_t x_stride, const float *ts, const float *bias, void *y, int N, int K,
                    int T, int y_dtype, int *status, bool early, cudaStream_t st) {
    GemmArgs a{};
    a.cs = cs; a.ts = ts; a.bias = bias; a.y = y; a.status = status; a.N = N; a.T = T; a.steps = (K + kStep - 1) / kStep;
    a.y_dtype = y_dtype; a.early = early;
    a.vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & (y_dtype == JQ_F32 ? 15u : 7u)) == 0;
    const int64_t ws = jq_row_stride_codes(K);
    if (T <= 16) return launch<16>(a, w, ws, x, x_stride, K, st);
    if (T <= 32) return launch<32>(a, w, ws, x, x_stride, K, st);
    if (T <= 64) return launch<64>(a, w, ws, x, x_stride, K, st);
    if (T <= 128) return launch<128>(a, w, ws, x, x_stride, K, st);
    return launch<256>(a, w, ws, x, x_stride, K, st);
}

static int check(const void *w, const float *cs, const void *y, const int *status, int N, int K, int B, int y_dtype) {
    if (!w || !cs || !y || !status) return JQ_ERR_NULL_PTR;
    if (N <= 0 || K <= 0 || B <= 0 || K > JQ_INT8_MAX_K) return JQ_ERR_BAD_SHAPE;
    if ((B + 255) / 256 > 65535) return JQ_ERR_BAD_SHAPE;
    if (y_dtype < 0 || y_dtype > 2) return JQ_ERR_BAD_DTYPE;
    const uintptr_t off = reinterpret_cast<uintptr_t>(y) & (y_dtype == JQ_F32 ? 3u : 1u);
    return !jq_aligned16(w) || (reinterpret_cast<uintptr_t>(cs) & 3u) || off ? JQ_ERR_BAD_ALIGN : JQ_OK;
}

static size_t scale_room(int rows) { return ((size_t)rows * 4 + 255) / 256 * 256; }

}  // namespace jq8

using namespace jq8;

extern "C" size_t jq_int8_scratch_bytes(int B, int K) {
    if (B <= 0 || K <= 0) return 0;
    return scale_room(B) + (size_t)B * jq_row_stride_codes(K);
}

extern "C" int jq_int8_linear(const void *qweight, const float *scales, const void *x, const float *bias, void *y, int N, int K, int B,
                              int had_block, int x_dtype, int y_dtype, void *scratch, size_t scratch_size, int *status, jq_stream_t stream) {
    if (!x || !scratch) return JQ_ERR_NULL_PTR;
    int rc = check(qweight, scales, y, status, N, K, B, y_dtype);
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
    const int rc = check(qweight, scales, y, status, N, K, B, y_dtype);
    if (rc) return rc;
    if (code_stride < K) return JQ_ERR_BAD_SHAPE;
    if (!jq_aligned16(codes) || code_stride % 16) return JQ_ERR_BAD_ALIGN;
    return multiply(qweight, scales, codes, code_stride, row_scales, bias, y, N, K, B, y_dtype, status, false, reinterpret_cast<cudaStream_t>(stream));
}
