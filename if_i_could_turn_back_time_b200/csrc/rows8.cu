// Activations as rows of 8-bit integers (sm_100a).
#include "rows8.cuh"

namespace jq8 {

struct QuantArgs {
    const void *x;
    long long stride_x, stride_q;      // between rows
    int8_t *codes;
    float *scales;
    int rows, width, parts;            // parts: CTAs of a cluster that share a row
    int inner;                         // around a row but the first and the last lie at least 16 elements of its neighbours
};

constexpr int kLong = 544;             // threads of a block of a cluster at most: eight of them hold JQ_INT8_MAX_K values

// What becomes of a row
enum Mode {
    kStraight,    // rows of 16-byte pieces, kept as they are, the maximum found in pairs of 16 bits
    kRotated,     // the same rows rotated: a thread's chunks are neighbours, so that less of the rotation crosses lanes
    kAnywhere     // rows that begin anywhere
};

// Blocks that an SM is to hold.  Both sides, us: 8191 x 11008 rotated, 74 with four and 68 with three; 8191 x 11007, 82 and 96; 20000 x 1024 rotated, a
// warp per row, 16 with four and 18 unbounded.
constexpr int blocks_of(int threads, bool rotated) { return threads == 0 ? 4 : threads == 384 ? (rotated ? 3 : 4) : threads == 512 ? 2 : 1; }

// A warp (kThreads 0), a block or a cluster of blocks per row, which stays in registers between its maximum and its codes.
// 8191 x 11008 bf16: 53 us straight (5.1 TB/s), 68 rotated, where instructions bind (17 per value: seven additions, two shuffles, four of
// encoding; issue slots 65 % busy, the L1 71 %; with a thread's chunks apart and the stages' sums one by one 100), 82 at 11007 values, where pieces
// are read twice and shifted (by elements 167).  64 x 8192: 2.8 us, nearly all of it the launch and two barriers.
template <class T, int kChunks, int kThreads, Mode kMode>
__global__ void __launch_bounds__(kThreads ? kThreads : 256, blocks_of(kThreads, kMode == kRotated)) quantize_kernel(const __grid_constant__ QuantArgs p) {
    constexpr bool kBlock = kThreads != 0;
    __shared__ Shared sh;
    __shared__ uint32_t s_top;
    jqta::pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int threads = kBlock ? blockDim.x : 32;
    const int row = kBlock ? blockIdx.y : blockIdx.x * 8 + (threadIdx.x >> 5);
    const int me = kBlock ? threadIdx.x : lane, part = kBlock ? blockIdx.x : 0;
    if (row >= p.rows) return;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.stride_x;
    int8_t *codes = p.codes + row * p.stride_q;
    Joined<kBlock> joined(sh);
    // the row's maximum, over the CTAs that share it too; the scale told once
    auto coder_of = [&](uint32_t m) {
        m = joined.top(m);
        if (kThreads == kLong) {
            if (me == 0) s_top = m;
            jqta::cluster_sync();
            for (int r = 0; r < p.parts; ++r) {
                uint32_t o;
                asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %1, %2; ld.shared::cluster.u32 %0, [a]; }" : "=r"(o) : "r"(jqta::smem_u32(&s_top)), "r"(r) : "memory");
                m = max(m, o);
            }
            jqta::cluster_sync();                 // (nobody leaves while another reads)
        }
        const Coder coder(m);
        if (me == 0 && part == 0) p.scales[row] = coder.told();
        return coder;
    };
    if constexpr (kMode == kStraight) {
        const int c0 = part * threads * kChunks + me;
        Held<kPieces, T> held[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) held[j].load(x, (c0 + j * threads) * 8, p.width);
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = max(m, largest_bits(held[j].raw));
        } else {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = __vmaxu2(m, largest_pair(held[j].raw));
            m = bits_of_pair(m, T());
        }
        const Coder coder = coder_of(m);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float v[8];
            held[j].get(v);
            coder.template store_as<kPieces>(codes, (c0 + j * threads) * 8, p.width, v);
        }
    } else if constexpr (kMode == kRotated) {
        const int c0 = (part * threads + me) * kChunks, i = c0 * 8;
        float v[kChunks][8];
        Held<kPieces, T> held[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) held[j].load(x, i + 8 * j, p.width);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) held[j].get(v[j]);
        rotate128<kChunks>(v, lane);
        const Coder coder = coder_of(largest_rotated(v));
        if (i < p.width) {
            if constexpr (kChunks == 1) {
                *reinterpret_cast<uint2 *>(codes + i) = coder.eight(v[0]);
            } else {
#pragma unroll
                for (int j = 0; j < kChunks; j += 2) {
                    const uint2 a = coder.eight(v[j]), b = coder.eight(v[j + 1]);
                    *reinterpret_cast<uint4 *>(codes + i + 8 * j) = make_uint4(a.x, a.y, b.x, b.y);
                }
            }
        }
    } else {
        const int c0 = part * threads * kChunks + me;
        const bool near = p.inner && row > 0 && row + 1 < p.rows;
        Raw8<T> raw[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = load_anywhere(x, c0 + j * threads, p.width, near);
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = max(m, largest_bits(raw[j]));
        } else {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = __vmaxu2(m, largest_pair(raw[j]));
            m = bits_of_pair(m, T());
        }
        const Coder coder = coder_of(m);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float v[8];
            widen(raw[j], v);
            coder.store(codes, (c0 + j * threads) * 8, p.width, v);
        }
    }
}

struct DequantArgs {
    const int8_t *codes;
    const float *scales;
    void *out;
    long long stride_q;
    int rows, width, segments;
};

// A warp per 1024 values of a row.
template <class T, bool kVec>
__global__ void __launch_bounds__(256) dequantize_kernel(const __grid_constant__ DequantArgs p) {
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const long long row = unit / p.segments;
    if (row >= p.rows) return;
    const int seg = (int)(unit % p.segments);
    const int8_t *codes = p.codes + row * p.stride_q;
    T *out = reinterpret_cast<T *>(p.out) + row * p.width;
    const float s = p.scales[row];
    if constexpr (kVec) {
        uint2 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = (seg * 128 + 32 * j + lane) * 8;
            q[j] = i < p.width ? *reinterpret_cast<const uint2 *>(codes + i) : make_uint2(0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)((k < 4 ? q[j].x : q[j].y) >> 8 * (k & 3)) * s;
            store_chunk<kPieces>(out, (seg * 128 + 32 * j + lane) * 8, p.width, v);
        }
    } else {
        // chunks that are 16-byte pieces of the output: `off` elements behind, so that their codes lie across two words of eight
        const int off = (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) & 7);
        auto eight = [&](int at) -> uint64_t { return at >= 0 && at + 8 <= p.width ? *reinterpret_cast<const uint64_t *>(codes + at) : 0ull; };
#pragma unroll 2
        for (int j = 0; j < 4; ++j) {
            const int c = seg * 128 + 32 * j + lane, i = c * 8 - off;
            if (i >= 0 && c * 8 + 8 <= p.width) {
                uint64_t q = eight(c * 8);
                if (off) q = q << 8 * off | eight(c * 8 - 8) >> (64 - 8 * off);
                alignas(16) T e[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = (T)((float)(int8_t)(q >> 8 * k) * s);
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; ++k)
                    *reinterpret_cast<uint4 *>(reinterpret_cast<unsigned char *>(out + i) + 16 * k) = reinterpret_cast<const uint4 *>(e)[k];
            } else if (i < p.width) {
                for (int k = 0; k < 8; ++k)
                    if (i + k >= 0 && i + k < p.width) out[i + k] = (T)((float)codes[i + k] * s);
            }
        }
    }
}

// ---- host side -------------------------------------------------------------------------

static int launch_parts(void (*k)(const QuantArgs), const QuantArgs &a, const Cut &c, cudaStream_t st) {
    if (a.parts == 1) {
        k<<<c.threads ? dim3(1, a.rows) : dim3((a.rows + 7) / 8), c.threads ? c.threads : 256, 0, st>>>(a);
        return jq_launch_status();
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)a.parts, (unsigned)a.rows);
    cfg.blockDim = dim3((unsigned)c.threads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, k, a));
    return jq_launch_status();
}

template <class T>
static int launch_quantize(QuantArgs &a, bool vec, bool rotate, cudaStream_t st) {
    const int sms = jq_sm_count(), chunks = chunks_of(a.width, kPieces);
    Cut c = cut_of(chunks, a.rows, sms, 4);
    void (*k)(const QuantArgs);
    a.parts = 1;
    if (chunks > 4096) {
        // Longer rows than a block keeps go to clusters of eight blocks.  (Shorter ones in clusters, so that some blocks load while others
        // compute, were slower: 4096 x 28672 bf16 rotated 143 us in clusters of three, 121 in blocks of 896 threads.)
        a.parts = 8;
        c = Cut{4, ((chunks + 31) / 32 + 31) / 32 * 32};
        k = rotate ? quantize_kernel<T, 4, kLong, kRotated> : vec ? quantize_kernel<T, 4, kLong, kStraight> : quantize_kernel<T, 4, kLong, kAnywhere>;
    } else if (rotate) {
        k = c.threads == 0 ? (c.chunks == 1 ? quantize_kernel<T, 1, 0, kRotated> : c.chunks == 2 ? quantize_kernel<T, 2, 0, kRotated> : quantize_kernel<T, 4, 0, kRotated>)
                           : (c.chunks == 1 ? quantize_kernel<T, 1, 1024, kRotated> : c.threads <= 384 ? quantize_kernel<T, 4, 384, kRotated> : quantize_kernel<T, 4, 1024, kRotated>);
    } else if (vec && sizeof(T) == 2 && chunks > 1536 && a.rows > 2 * sms) {
        // (eight chunks a thread, so that an SM holds two blocks: 4096 x 28672 bf16 71 us, in one block of 896 threads 97)
        c = Cut{8, ((chunks + 7) / 8 + 31) / 32 * 32};
        k = quantize_kernel<T, 8, 512, kStraight>;
    } else if (vec) {
        k = c.threads == 0 ? (c.chunks == 1 ? quantize_kernel<T, 1, 0, kStraight> : c.chunks == 2 ? quantize_kernel<T, 2, 0, kStraight> :
                              c.chunks == 3 ? quantize_kernel<T, 3, 0, kStraight> : quantize_kernel<T, 4, 0, kStraight>)
                           : (c.chunks == 1 ? quantize_kernel<T, 1, 1024, kStraight> : c.threads <= 384 ? quantize_kernel<T, 4, 384, kStraight> : quantize_kernel<T, 4, 1024, kStraight>);
    } else {
        k = c.threads == 0 ? (c.chunks == 1 ? quantize_kernel<T, 1, 0, kAnywhere> : c.chunks == 2 ? quantize_kernel<T, 2, 0, kAnywhere> : quantize_kernel<T, 4, 0, kAnywhere>)
                           : (c.chunks == 1 ? quantize_kernel<T, 1, 1024, kAnywhere> : c.threads <= 384 ? quantize_kernel<T, 4, 384, kAnywhere> : quantize_kernel<T, 4, 1024, kAnywhere>);
    }
    if (c.threads && a.rows > 65535) {
        // rows are the grid's second dimension: in parts of it
        for (long long r0 = 0; r0 < a.rows; r0 += 65535) {
            QuantArgs b = a;
            b.rows = a.rows - r0 < 65535 ? (int)(a.rows - r0) : 65535;
            b.x = reinterpret_cast<const T *>(a.x) + r0 * a.stride_x;
            b.codes += r0 * a.stride_q;
            b.scales += r0;
            const int rc = launch_parts(k, b, c, st);
            if (rc) return rc;
        }
        return JQ_OK;
    }
    return launch_parts(k, a, c, st);
}

}  // namespace jq8

using namespace jq8;

extern "C" int jq_quantize_rows(const void *x, int64_t row_stride, int rows, int K, int had_block, int x_dtype, void *codes,
                                int64_t code_stride, float *scales, jq_stream_t stream) {
    if (!x || !codes || !scales) return JQ_ERR_NULL_PTR;
    if (rows <= 0 || rows > JQ_INT8_MAX_ROWS || K <= 0 || K > JQ_INT8_MAX_K || code_stride < K || row_stride < 0) return JQ_ERR_BAD_SHAPE;
    if (had_block != 0 && (had_block != 128 || K % 128)) return JQ_ERR_BAD_SHAPE;
    if (x_dtype < 0 || x_dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (!jq_aligned16(codes) || code_stride % 16) return JQ_ERR_BAD_ALIGN;
    const int size = x_dtype == JQ_F32 ? 4 : 2;
    if (!jq_whole(x, size) || !jq_whole(scales, 4)) return JQ_ERR_BAD_ALIGN;
    QuantArgs a{};
    a.x = x; a.stride_x = row_stride; a.stride_q = code_stride;
    a.codes = reinterpret_cast<int8_t *>(codes); a.scales = scales;
    a.rows = rows; a.width = K; a.inner = K >= 16 && row_stride >= K;
    const bool vec = K % 8 == 0 && aligned(x, row_stride, size);
    if (had_block && !vec) return JQ_ERR_BAD_ALIGN;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x_dtype == JQ_F32) return launch_quantize<float>(a, vec, had_block != 0, st);
    if (x_dtype == JQ_F16) return launch_quantize<__half>(a, vec, had_block != 0, st);
    return launch_quantize<__nv_bfloat16>(a, vec, had_block != 0, st);
}

extern "C" int jq_dequantize_rows(const void *codes, int64_t code_stride, const float *scales, int rows, int K, void *out, int dtype,
                                  jq_stream_t stream) {
    if (!codes || !scales || !out) return JQ_ERR_NULL_PTR;
    if (rows <= 0 || rows > JQ_INT8_MAX_ROWS || K <= 0 || K > JQ_INT8_MAX_K || code_stride < K) return JQ_ERR_BAD_SHAPE;
    if (dtype < 0 || dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (!jq_aligned16(codes) || code_stride % 16 || !jq_whole(scales, 4) || !jq_whole(out, dtype == JQ_F32 ? 4 : 2)) return JQ_ERR_BAD_ALIGN;
    DequantArgs a{};
    a.codes = reinterpret_cast<const int8_t *>(codes); a.scales = scales; a.out = out; a.stride_q = code_stride;
    a.rows = rows; a.width = K;
    const bool vec = K % 8 == 0 && jq_aligned16(out);
    a.segments = (K + (vec ? 0 : 7) + 1023) / 1024;
    const long long blocks = ((long long)rows * a.segments + 7) / 8;
    if (blocks > 0x7fffffff) return JQ_ERR_BAD_SHAPE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    void (*const kernels[3][2])(const DequantArgs) = {{dequantize_kernel<float, false>, dequantize_kernel<float, true>},
                                                      {dequantize_kernel<__half, false>, dequantize_kernel<__half, true>},
                                                      {dequantize_kernel<__nv_bfloat16, false>, dequantize_kernel<__nv_bfloat16, true>}};
    kernels[dtype][vec]<<<(unsigned)blocks, 256, 0, st>>>(a);
    return jq_launch_status();
}
