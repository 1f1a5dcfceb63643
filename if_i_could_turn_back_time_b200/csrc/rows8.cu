// Activations as rows of 8-bit integers (sm_100a).
#include "rows8.cuh"

namespace jq8 {

struct QuantArgs {
    const void *x;
    long long stride_x, stride_q;      // between rows
    int8_t *codes;
    float *scales;
    int rows, width, rotate, neighbours, vec;
};

// How a thread's chunks lie and what becomes of them
enum Mode {
    kStraight,    // rows of 16-byte pieces, not rotated: kept as they are, the maximum found in pairs of 16 bits
    kRotated,     // rotated: a thread's chunks are neighbours, so that less of the rotation crosses lanes
    kGeneral,     // any width, alignment and stride, rotated or not
    kTiled        // the same for rows that a block does not keep, which are read twice
};

// A warp (kThreads 0) or a block per row, which stays in registers between its maximum and its codes.
template <class T, int kChunks, int kThreads, Mode kMode>
__global__ void __launch_bounds__(kThreads ? kThreads : 256) quantize_kernel(const __grid_constant__ QuantArgs p) {
    constexpr bool kBlock = kThreads != 0;
    __shared__ Shared sh;
    jqta::pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int threads = kBlock ? blockDim.x : 32, me = kBlock ? threadIdx.x : lane;
    const int row = kBlock ? blockIdx.x : blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.stride_x;
    int8_t *codes = p.codes + row * p.stride_q;
    Joined<kBlock> joined(sh);
    if constexpr (kMode == kStraight) {
        const Places at(p.width, true);
        Raw8<T> raw[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = load_chunk(x, me + j * threads, at, true);
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = max(m, largest_bits(raw[j]));
        } else {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = __vmaxu2(m, largest_pair(raw[j]));
            m = bits_of_pair(m, T());
        }
        const Coder coder(joined.top(m));
        if (me == 0) p.scales[row] = coder.told();
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int i = (me + j * threads) * 8;
            float v[8];
            widen(raw[j], v);
            if (i < p.width) *reinterpret_cast<uint2 *>(codes + i) = coder.eight(v);
        }
    } else if constexpr (kMode == kRotated) {
        const Places at(p.width, true);
        float v[kChunks][8];
        Raw8<T> raw[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = load_chunk(x, me * kChunks + j, at, true);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) widen(raw[j], v[j]);
        rotate128<kChunks>(v, lane);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) m = max(m, largest_bits(v[j]));
        const Coder coder(joined.top(m));
        if (me == 0) p.scales[row] = coder.told();
        const int i = me * kChunks * 8;
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
        const Places at(p.width, p.neighbours);
        const int tile = threads * kChunks, chunks = p.neighbours ? (p.width + 7) / 8 : (p.width + 255) / 256 * 32;
        const int end = kMode == kTiled ? chunks : 1;
        float v[kChunks][8];
        auto read = [&](int c0) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float one[1][8];
                widen(load_chunk(x, c0 + me + j * threads, at, p.vec), one[0]);
                if (p.rotate) rotate128<1>(one, lane);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] = one[0][k];
            }
        };
        uint32_t m = 0;
        for (int c0 = 0; c0 < end; c0 += tile) {
            read(c0);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) m = max(m, largest_bits(v[j]));
        }
        const Coder coder(joined.top(m));
        if (me == 0) p.scales[row] = coder.told();
        for (int c0 = 0; c0 < end; c0 += tile) {
            if (kMode == kTiled) read(c0);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) coder.store(codes, c0 + me + j * threads, at, v[j]);
        }
    }
}

struct DequantArgs {
    const int8_t *codes;
    const float *scales;
    void *out;
    long long stride_q;
    int rows, width, neighbours, vec, dtype, segments;
};

// A warp per 1024 values of a row.
template <class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const __grid_constant__ DequantArgs p) {
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const long long row = unit / p.segments;
    if (row >= p.rows) return;
    const int c0 = (int)(unit % p.segments) * 128 + lane;
    const Places at(p.width, p.neighbours);
    const int8_t *codes = p.codes + row * p.stride_q;
    T *out = reinterpret_cast<T *>(p.out) + row * p.width;
    const float s = p.scales[row];
    uint2 q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = at.first(c0 + 32 * j);
        q[j] = make_uint2(0, 0);
        if (at.next == 1) {
            if (i < at.width) q[j] = *reinterpret_cast<const uint2 *>(codes + i);
        } else {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + 32 * k < at.width) w[k >> 2] |= (uint32_t)(uint8_t)codes[i + 32 * k] << 8 * (k & 3);
            q[j] = make_uint2(w[0], w[1]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)((k < 4 ? q[j].x : q[j].y) >> 8 * (k & 3)) * s;
        store_chunk(out, c0 + 32 * j, at, p.vec, v);
    }
}

// ---- host side -------------------------------------------------------------------------

template <class T>
static int launch_quantize(const QuantArgs &a, cudaStream_t st) {
    const int sms = jq_sm_count();
    void (*k)(const QuantArgs);
    Cut c;
    if (a.vec && a.width <= kMostKept) {
        c = cut_of(a.width, true, a.rows, sms, 4);
        if (a.rotate) {
            // (chunks that are neighbours: one, or four, which a row of 128 always fills)
            if (c.threads == 0) c.chunks = c.chunks == 1 ? 1 : 4;
            k = c.threads == 0 ? (c.chunks == 1 ? quantize_kernel<T, 1, 0, kRotated> : quantize_kernel<T, 4, 0, kRotated>)
                               : (c.chunks == 1 ? quantize_kernel<T, 1, 1024, kRotated> : c.threads <= 512 ? quantize_kernel<T, 4, 512, kRotated> : quantize_kernel<T, 4, 1024, kRotated>);
        } else {
            k = c.threads == 0 ? (c.chunks == 1 ? quantize_kernel<T, 1, 0, kStraight> : c.chunks == 2 ? quantize_kernel<T, 2, 0, kStraight> :
                                  c.chunks == 3 ? quantize_kernel<T, 3, 0, kStraight> : quantize_kernel<T, 4, 0, kStraight>)
                               : (c.chunks == 1 ? quantize_kernel<T, 1, 1024, kStraight> : quantize_kernel<T, 4, 1024, kStraight>);
        }
    } else {
        c = cut_of(a.width, a.neighbours, a.rows, sms, 4);
        const int chunks = a.neighbours ? a.width / 8 : (a.width + 255) / 256 * 32;
        if (c.threads == 0) k = quantize_kernel<T, 4, 0, kGeneral>;
        else if (c.threads * c.chunks < chunks) k = quantize_kernel<T, 4, 1024, kTiled>;
        else k = c.chunks == 1 ? quantize_kernel<T, 1, 1024, kGeneral> : quantize_kernel<T, 4, 1024, kGeneral>;
    }
    k<<<c.threads ? a.rows : (a.rows + 7) / 8, c.threads ? c.threads : 256, 0, st>>>(a);
    return jq_launch_status();
}

}  // namespace jq8

using namespace jq8;

extern "C" int jq_quantize_rows(const void *x, int64_t row_stride, int rows, int K, int had_block, int x_dtype, void *codes,
                                int64_t code_stride, float *scales, jq_stream_t stream) {
    if (!x || !codes || !scales) return JQ_ERR_NULL_PTR;
    if (rows <= 0 || K <= 0 || K > JQ_INT8_MAX_K || code_stride < K || row_stride < 0) return JQ_ERR_BAD_SHAPE;
    if (had_block != 0 && (had_block != 128 || K % 128)) return JQ_ERR_BAD_SHAPE;
    if (x_dtype < 0 || x_dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (!jq_aligned16(codes) || code_stride % 16) return JQ_ERR_BAD_ALIGN;
    const int size = x_dtype == JQ_F32 ? 4 : 2;
    QuantArgs a{};
    a.x = x; a.stride_x = row_stride; a.stride_q = code_stride;
    a.codes = reinterpret_cast<int8_t *>(codes); a.scales = scales;
    a.rows = rows; a.width = K; a.rotate = had_block != 0;
    a.neighbours = K % 8 == 0;
    a.vec = a.neighbours && aligned(x, row_stride, size);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x_dtype == JQ_F32) return launch_quantize<float>(a, st);
    if (x_dtype == JQ_F16) return launch_quantize<__half>(a, st);
    return launch_quantize<__nv_bfloat16>(a, st);
}

extern "C" int jq_dequantize_rows(const void *codes, int64_t code_stride, const float *scales, int rows, int K, void *out, int dtype,
                                  jq_stream_t stream) {
    if (!codes || !scales || !out) return JQ_ERR_NULL_PTR;
    if (rows <= 0 || K <= 0 || code_stride < K) return JQ_ERR_BAD_SHAPE;
    if (dtype < 0 || dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (!jq_aligned16(codes) || code_stride % 16) return JQ_ERR_BAD_ALIGN;
    DequantArgs a{};
    a.codes = reinterpret_cast<const int8_t *>(codes); a.scales = scales; a.out = out; a.stride_q = code_stride;
    a.rows = rows; a.width = K; a.neighbours = K % 8 == 0; a.dtype = dtype;
    a.vec = a.neighbours && jq_aligned16(out);
    a.segments = (K + 1023) / 1024;
    const long long blocks = ((long long)rows * a.segments + 7) / 8;
    if (blocks > 0x7fffffff) return JQ_ERR_BAD_SHAPE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == JQ_F32) dequantize_kernel<float><<<(unsigned)blocks, 256, 0, st>>>(a);
    else if (dtype == JQ_F16) dequantize_kernel<__half><<<(unsigned)blocks, 256, 0, st>>>(a);
    else dequantize_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, st>>>(a);
    return jq_launch_status();
}
