// Activations as rows of 8-bit integers, and the norms around a block, which can write them (sm_100a).
#include "rows8.cuh"

namespace jq8 {

constexpr int kMostKept = 32768;       // longest row that a block keeps in registers: 1024 threads with four chunks of eight values

struct QuantArgs {
    const void *x;
    long long stride_x, stride_q;      // between rows
    int8_t *codes;
    float *scales;
    int rows, width, rotate, neighbours, vec;
};

// A warp or a block per row, which it keeps in registers between finding its maximum and writing its codes (kTiled: longer rows, read
// twice).
template <class T, int kChunks, bool kBlock, bool kTiled>
__global__ void __launch_bounds__(kBlock ? 1024 : 256) quantize_kernel(const __grid_constant__ QuantArgs p) {
    __shared__ Shared sh;
    jqta::pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int threads = kBlock ? blockDim.x : 32, me = kBlock ? threadIdx.x : lane;
    const int row = kBlock ? blockIdx.x : blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.stride_x;
    int8_t *codes = p.codes + row * p.stride_q;
    const Places at(p.width, p.neighbours);
    const int tile = threads * kChunks, chunks = p.neighbours ? (p.width + 7) / 8 : (p.width + 255) / 256 * 32;
    Joined<kBlock> joined(sh);
    float v[kChunks][8];
    auto read = [&](int c0) {
        Raw8<T> raw[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = load_chunk(x, c0 + me + j * threads, at, p.vec);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            widen(raw[j], v[j]);
            if (p.rotate) rotate128(v[j], lane);
        }
    };
    uint32_t m = 0;
    for (int c0 = 0; c0 < (kTiled ? chunks : 1); c0 += tile) {
        read(c0);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) m = max(m, largest_bits(v[j]));
    }
    const Coder coder(joined.top(m));
    if (me == 0) p.scales[row] = coder.told();
    for (int c0 = 0; c0 < (kTiled ? chunks : 1); c0 += tile) {
        if (kTiled) read(c0);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) coder.store(codes, c0 + me + j * threads, at, v[j]);
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

struct NormArgs {
    const void *x, *residual;          // residual: null for none
    void *r, *h;                       // r: null where it is x itself; h: values of x's type, or null
    int8_t *codes;                     // with scales, in h's place
    float *scales;
    const void *weight, *bias, *post_weight, *post_bias, *gate;
    long long stride_x, stride_res, stride_q;
    long long gate_outer, gate_inner;  // gate of row i: at (i / inner) gate_outer + (i % inner) gate_inner
    int inner, gate_one;               // gate_one: one value for the whole row
    int rows, width;
    float scale, eps;
    int layer, post, rotate, neighbours;
    int wdtype, gdtype;                // types of the four vectors and of the gate
    int vec_x, vec_res, vec_r, vec_h, vec_w, vec_g;
};

// A warp or a block per row, which stays in registers from the first read to the last write:
//   u = N(x) post_weight + post_bias (or x),  r = residual + scale * (gate * u),  h = N(r) weight + bias,
// N(v) = v / sqrt(mean(v^2) + eps), or of v - mean(v).  All in fp32; h follows from r as it was before its rounding.
template <class T, class R, int kChunks, bool kBlock>
__global__ void __launch_bounds__(kBlock ? 1024 : 256) norm_kernel(const __grid_constant__ NormArgs p) {
    __shared__ Shared sh;
    jqta::pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int threads = kBlock ? blockDim.x : 32, me = kBlock ? threadIdx.x : lane;
    const int row = kBlock ? blockIdx.x : blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const Places at(p.width, p.neighbours);
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.stride_x;
    Joined<kBlock> joined(sh);
    const float each = 1.f / (float)p.width;
    float v[kChunks][8];
    Raw8<R> res[kChunks];
    {
        Raw8<T> raw[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = load_chunk(x, me + j * threads, at, p.vec_x);
        if (p.residual) {
            const R *from = reinterpret_cast<const R *>(p.residual) + row * p.stride_res;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) res[j] = load_chunk(from, me + j * threads, at, p.vec_res);
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j) widen(raw[j], v[j]);
    }
    // whether element k of chunk j is one of the row
    auto in = [&](int j, int k) { return at.first(me + j * threads) + k * at.next < at.width; };
    auto normed = [&](const void *weight, const void *bias) {
        float mean = 0.f, s = 0.f;
        if (p.layer) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) mean += v[j][k];                       // (zeros behind the row's end)
            mean = joined.sum(mean) * each;
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] = in(j, k) ? v[j][k] - mean : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) s = fmaf(v[j][k], v[j][k], s);
        s = rsqrtf(joined.sum(s) * each + p.eps);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float w[8], b[8];
            if (weight) load_any(weight, p.wdtype, me + j * threads, at, p.vec_w, w);
            if (bias) load_any(bias, p.wdtype, me + j * threads, at, p.vec_w, b);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[j][k] *= s;
                if (weight) v[j][k] *= w[k];
                if (bias) v[j][k] += b[k];
            }
        }
    };
    if (p.post) normed(p.post_weight, p.post_bias);
    if (p.gate) {
        const long long g0 = (long long)(row / p.inner) * p.gate_outer + (long long)(row % p.inner) * p.gate_inner;
        const void *gate = reinterpret_cast<const unsigned char *>(p.gate) + g0 * (p.gdtype == JQ_F32 ? 4 : 2);
        const float one = p.gate_one ? jq::load_act(gate, 0, p.gdtype) : 0.f;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float g[8];
            if (!p.gate_one) load_any(gate, p.gdtype, me + j * threads, at, p.vec_g, g);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] *= p.gate_one ? one : g[k];
        }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        float old[8];
        if (p.residual) widen(res[j], old);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[j][k] *= p.scale;
            if (p.residual) v[j][k] += old[k];
        }
    }
    if (p.r) {
        R *r = reinterpret_cast<R *>(p.r) + (long long)row * p.width;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) store_chunk(r, me + j * threads, at, p.vec_r, v[j]);
    }
    // a post bias or an infinite gate leaves values behind the row's end
    if (p.post_bias || p.gate)
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] = in(j, k) ? v[j][k] : 0.f;
    normed(p.weight, p.bias);
    if (!p.codes) {
        T *h = reinterpret_cast<T *>(p.h) + (long long)row * p.width;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) store_chunk(h, me + j * threads, at, p.vec_h, v[j]);
        return;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        if (p.rotate) rotate128(v[j], lane);
        if (!p.neighbours || me + j * threads < p.width / 8) {
#pragma unroll
            for (int k = 0; k < 8; ++k) m = max(m, in(j, k) ? __float_as_uint(v[j][k]) & 0x7fffffffu : 0u);
        }
    }
    const Coder coder(joined.top(m));
    if (me == 0) p.scales[row] = coder.told();
    int8_t *codes = p.codes + row * p.stride_q;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) coder.store(codes, me + j * threads, at, v[j]);
}

// ---- host side -------------------------------------------------------------------------

struct Cut { int chunks, threads; };   // threads 0: a warp per row

// A row's chunks over threads.  Up to 128 chunks a warp has them all and needs no barrier; longer rows have a block, with four chunks
// per thread (loads in flight together, few warps at the barriers) unless rows are so few that latency counts: then one.
static Cut cut_of(int width, bool neighbours, int rows, int sms) {
    const int chunks = neighbours ? (width + 7) / 8 : (width + 255) / 256 * 32;
    if (chunks <= 128 && (rows > 2 * sms || chunks <= 32)) return Cut{chunks <= 32 ? 1 : (chunks <= 64 ? 2 : 4), 0};
    int per = rows > 2 * sms ? 4 : 1;
    while ((chunks + per - 1) / per > 1024 && per < 4) per *= 2;
    int threads = ((chunks + per - 1) / per + 31) / 32 * 32;
    return Cut{per, threads < 1024 ? threads : 1024};
}

static bool aligned(const void *p, long long stride, int size) {
    return jq_aligned16(p) && stride * size % 16 == 0;
}

template <class T>
static int launch_quantize(const QuantArgs &a, const Cut &c, bool tiled, cudaStream_t st) {
    void (*k)(const QuantArgs);
    if (tiled) k = quantize_kernel<T, 4, true, true>;
    else if (c.threads == 0) k = c.chunks == 1 ? quantize_kernel<T, 1, false, false> : (c.chunks == 2 ? quantize_kernel<T, 2, false, false> : quantize_kernel<T, 4, false, false>);
    else k = c.chunks == 1 ? quantize_kernel<T, 1, true, false> : (c.chunks == 2 ? quantize_kernel<T, 2, true, false> : quantize_kernel<T, 4, true, false>);
    k<<<c.threads ? a.rows : (a.rows + 7) / 8, c.threads ? c.threads : 256, 0, st>>>(a);
    return jq_launch_status();
}

template <class T, class R>
static int launch_norm(const NormArgs &a, const Cut &c, cudaStream_t st) {
    void (*k)(const NormArgs);
    if (c.threads == 0) k = c.chunks == 1 ? norm_kernel<T, R, 1, false> : (c.chunks == 2 ? norm_kernel<T, R, 2, false> : norm_kernel<T, R, 4, false>);
    else k = c.chunks == 1 ? norm_kernel<T, R, 1, true> : (c.chunks == 2 ? norm_kernel<T, R, 2, true> : norm_kernel<T, R, 4, true>);
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
    const Cut c = cut_of(K, a.neighbours, rows, jq_sm_count());
    const int chunks = a.neighbours ? K / 8 : (K + 255) / 256 * 32;
    const bool tiled = c.threads != 0 && c.threads * c.chunks < chunks;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x_dtype == JQ_F32) return launch_quantize<float>(a, c, tiled, st);
    if (x_dtype == JQ_F16) return launch_quantize<__half>(a, c, tiled, st);
    return launch_quantize<__nv_bfloat16>(a, c, tiled, st);
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

extern "C" int jq_residual_norm(const jq_norm *n, jq_stream_t stream) {
    if (!n || !n->x || (!n->h && !n->codes) || (n->codes && !n->scales)) return JQ_ERR_NULL_PTR;
    if (n->rows <= 0 || n->width <= 0 || n->width > kMostKept || n->stride_x < 0 || n->stride_residual < 0) return JQ_ERR_BAD_SHAPE;
    if (n->kind != JQ_NORM_RMS && n->kind != JQ_NORM_LAYER) return JQ_ERR_UNSUPPORTED;
    if (n->had_block != 0 && (n->had_block != 128 || n->width % 128 || !n->codes)) return JQ_ERR_BAD_SHAPE;
    if (n->gate && n->gate_inner_rows <= 0) return JQ_ERR_BAD_SHAPE;
    const int types[4] = {n->x_dtype, n->residual_dtype, n->weight_dtype, n->gate_dtype};
    for (int t : types)
        if (t < 0 || t > 2) return JQ_ERR_BAD_DTYPE;
    if (n->residual_dtype != n->x_dtype && n->residual_dtype != JQ_F32) return JQ_ERR_BAD_DTYPE;
    if (n->codes && (!jq_aligned16(n->codes) || n->stride_codes % 16)) return JQ_ERR_BAD_ALIGN;
    if (n->codes && n->stride_codes < n->width) return JQ_ERR_BAD_SHAPE;
    const int W = n->width, xs = n->x_dtype == JQ_F32 ? 4 : 2, rs = n->residual_dtype == JQ_F32 ? 4 : 2;
    NormArgs a{};
    a.x = n->x; a.residual = n->residual; a.r = n->r; a.h = n->h; a.codes = reinterpret_cast<int8_t *>(n->codes); a.scales = n->scales;
    a.weight = n->weight; a.bias = n->bias; a.post_weight = n->post_weight; a.post_bias = n->post_bias; a.gate = n->gate;
    a.stride_x = n->stride_x; a.stride_res = n->stride_residual; a.stride_q = n->stride_codes;
    a.gate_outer = n->gate_outer; a.gate_inner = n->gate_inner; a.inner = n->gate ? n->gate_inner_rows : 1; a.gate_one = n->gate_one;
    a.rows = n->rows; a.width = W; a.scale = n->scale; a.eps = n->eps;
    a.layer = n->kind == JQ_NORM_LAYER; a.post = n->post; a.rotate = n->had_block != 0;
    a.wdtype = n->weight_dtype; a.gdtype = n->gate_dtype;
    a.neighbours = W % 8 == 0;
    if (a.neighbours) {
        const int ws = n->weight_dtype == JQ_F32 ? 4 : 2, gs = n->gate_dtype == JQ_F32 ? 4 : 2;
        a.vec_x = aligned(n->x, n->stride_x, xs);
        a.vec_res = n->residual && aligned(n->residual, n->stride_residual, rs);
        a.vec_r = jq_aligned16(n->r); a.vec_h = jq_aligned16(n->h);
        a.vec_w = aligned(n->weight, 0, ws) && aligned(n->bias, 0, ws) && aligned(n->post_weight, 0, ws) && aligned(n->post_bias, 0, ws);
        a.vec_g = aligned(n->gate, n->gate_outer, gs) && n->gate_inner * gs % 16 == 0;
    }
    const Cut c = cut_of(W, a.neighbours, n->rows, jq_sm_count());
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (n->x_dtype == JQ_F32) return launch_norm<float, float>(a, c, st);
    if (n->x_dtype == JQ_F16) return n->residual_dtype == JQ_F32 ? launch_norm<__half, float>(a, c, st) : launch_norm<__half, __half>(a, c, st);
    return n->residual_dtype == JQ_F32 ? launch_norm<__nv_bfloat16, float>(a, c, st) : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, c, st);
}
