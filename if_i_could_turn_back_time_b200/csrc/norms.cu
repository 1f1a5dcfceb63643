// The norms around a block with its gate and residual sum (sm_100a).
#include "rows8.cuh"

namespace jq8 {

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
    int vec_x, vec_res, vec_r, vec_h, vec_w, vec_g, wide_w, wide_g;
};

// Eight values of a vector of T or of fp32, as they lie (weights: the same for every row, so that they come from the caches)
template <class T> struct Weights {
    uint4 a, b;
    __device__ __forceinline__ void load(const void *p, bool wide, int i, int width) {
        a = b = make_uint4(0, 0, 0, 0);
        if (i >= width) return;
        const uint4 *from = reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned char *>(p) + (size_t)i * (wide ? 4 : sizeof(T)));
        a = from[0];
        if (wide) b = from[1];
    }
    __device__ __forceinline__ void get(bool wide, float (&v)[8]) const {
        if (wide) {
            Raw8<float> r;
            r.w[0] = a; r.w[1] = b;
            widen(r, v);
        } else if constexpr (sizeof(T) == 2) {
            Raw8<T> r;
            r.w[0] = a;
            widen(r, v);
        }
    }
};

// A warp (kThreads 0) or a block per row, which stays in registers from the first read to the last write:
//   u = N(x) post_weight + post_bias (or x),  r = residual + scale * (gate * u),  h = N(r) weight + bias,
// N(v) = v / sqrt(mean(v^2) + eps), or of v - mean(v).  All in fp32; h follows from r as it was before its rounding.
// kVec: every row and vector is of 16-byte pieces, and vectors are of T or fp32; the other form takes any width, alignment, stride and type.
template <class T, class R, int kChunks, int kThreads, bool kVec>
__global__ void __launch_bounds__(kThreads ? kThreads : 256) norm_kernel(const __grid_constant__ NormArgs p) {
    constexpr bool kBlock = kThreads != 0;
    __shared__ Shared sh;
    jqta::pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int threads = kBlock ? blockDim.x : 32, me = kBlock ? threadIdx.x : lane;
    const int row = kBlock ? blockIdx.x : blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const Places at(p.width, kVec || p.neighbours);
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.stride_x;
    Joined<kBlock> joined(sh);
    const float each = 1.f / (float)p.width;
    float v[kChunks][8];
    Raw8<R> res[kChunks];
    {
        Raw8<T> raw[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = load_chunk(x, me + j * threads, at, kVec || p.vec_x);
        if (p.residual) {
            const R *from = reinterpret_cast<const R *>(p.residual) + row * p.stride_res;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) res[j] = load_chunk(from, me + j * threads, at, kVec || p.vec_res);
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j) widen(raw[j], v[j]);
    }
    // whether element k of chunk j is one of the row
    auto in = [&](int j, int k) { return kVec ? (me + j * threads) * 8 < p.width : at.first(me + j * threads) + k * at.next < at.width; };
    auto vector = [&](const void *from, int j, float (&w)[8]) {           // of one of the four vectors
        if constexpr (kVec) {
            Weights<T> raw;
            raw.load(from, p.wide_w, (me + j * threads) * 8, p.width);
            raw.get(p.wide_w, w);
        } else {
            load_any(from, p.wdtype, me + j * threads, at, p.vec_w, w);
        }
    };
    auto normed = [&](const void *weight, const void *bias) {
        float s = 0.f;
        if (p.layer) {
            float mean = 0.f;
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
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] *= s;
        if (weight) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float w[8];
                vector(weight, j, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= w[k];
            }
        }
        if (bias) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float b[8];
                vector(bias, j, b);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] += b[k];
            }
        }
    };
    if (p.post) normed(p.post_weight, p.post_bias);
    float f = p.scale;
    if (p.gate) {
        const long long g0 = (long long)(row / p.inner) * p.gate_outer + (long long)(row % p.inner) * p.gate_inner;
        const void *gate = reinterpret_cast<const unsigned char *>(p.gate) + g0 * (p.gdtype == JQ_F32 ? 4 : 2);
        if (p.gate_one) {
            const float one = jq::load_act(gate, 0, p.gdtype);
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= one;
        } else {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float g[8];
                if constexpr (kVec) {
                    Weights<T> raw;
                    raw.load(gate, p.wide_g, (me + j * threads) * 8, p.width);
                    raw.get(p.wide_g, g);
                } else {
                    load_any(gate, p.gdtype, me + j * threads, at, p.vec_g, g);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= g[k];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        if (p.residual) {
            float old[8];
            widen(res[j], old);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] = old[k] + v[j][k] * f;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] *= f;
        }
    }
    if (p.r) {
        R *r = reinterpret_cast<R *>(p.r) + (long long)row * p.width;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) store_chunk(r, me + j * threads, at, kVec || p.vec_r, v[j]);
    }
    // (an infinite gate or root times the zeros behind the row's end is NaN)
    if (p.post || p.gate) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] = in(j, k) ? v[j][k] : 0.f;
    }
    normed(p.weight, p.bias);
    if (!p.codes) {
        T *h = reinterpret_cast<T *>(p.h) + (long long)row * p.width;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) store_chunk(h, me + j * threads, at, kVec || p.vec_h, v[j]);
        return;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        if (p.rotate) {
            float one[1][8];
#pragma unroll
            for (int k = 0; k < 8; ++k) one[0][k] = v[j][k];
            rotate128<1>(one, lane);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] = one[0][k];
        }
        m = max(m, largest_bits(v[j]));           // (zeros behind the row's end, or NaN where the row is NaN too)
    }
    const Coder coder(joined.top(m));
    if (me == 0) p.scales[row] = coder.told();
    int8_t *codes = p.codes + row * p.stride_q;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) coder.store(codes, me + j * threads, at, v[j]);
}

// ---- host side -------------------------------------------------------------------------

template <class T, class R>
static int launch_norm(const NormArgs &a, bool vec, cudaStream_t st) {
    const Cut c = cut_of(a.width, a.neighbours, a.rows, jq_sm_count(), 2);
    void (*k)(const NormArgs);
    if (vec) {
        if (c.threads == 0) k = c.chunks == 1 ? norm_kernel<T, R, 1, 0, true> : c.chunks == 2 ? norm_kernel<T, R, 2, 0, true> :
                                c.chunks == 3 ? norm_kernel<T, R, 3, 0, true> : norm_kernel<T, R, 4, 0, true>;
        else k = c.chunks == 1 ? norm_kernel<T, R, 1, 1024, true> : c.chunks == 2 ? norm_kernel<T, R, 2, 1024, true> : norm_kernel<T, R, 4, 1024, true>;
    } else {
        if (c.threads == 0) k = norm_kernel<T, R, 4, 0, false>;
        else k = c.chunks <= 2 ? norm_kernel<T, R, 2, 1024, false> : norm_kernel<T, R, 4, 1024, false>;
    }
    k<<<c.threads ? a.rows : (a.rows + 7) / 8, c.threads ? c.threads : 256, 0, st>>>(a);
    return jq_launch_status();
}

}  // namespace jq8

using namespace jq8;

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
    bool vec = false;
    if (a.neighbours) {
        const int gs = n->gate_dtype == JQ_F32 ? 4 : 2;
        const bool vectors = n->weight || n->bias || n->post_weight || n->post_bias;
        a.vec_x = aligned(n->x, n->stride_x, xs);
        a.vec_res = aligned(n->residual, n->stride_residual, rs);
        a.vec_r = jq_aligned16(n->r); a.vec_h = jq_aligned16(n->h);
        a.vec_w = jq_aligned16(n->weight) && jq_aligned16(n->bias) && jq_aligned16(n->post_weight) && jq_aligned16(n->post_bias);
        a.vec_g = n->gate_one || (aligned(n->gate, n->gate_outer, gs) && n->gate_inner * gs % 16 == 0);
        a.wide_w = n->weight_dtype == JQ_F32; a.wide_g = n->gate_dtype == JQ_F32;
        vec = a.vec_x && a.vec_res && a.vec_r && a.vec_h && a.vec_w && a.vec_g && (!vectors || n->weight_dtype == n->x_dtype || a.wide_w) &&
              (!n->gate || n->gate_one || n->gate_dtype == n->x_dtype || a.wide_g);
        a.vec_g = a.vec_g && !n->gate_one;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (n->x_dtype == JQ_F32) return launch_norm<float, float>(a, vec, st);
    if (n->x_dtype == JQ_F16) return n->residual_dtype == JQ_F32 ? launch_norm<__half, float>(a, vec, st) : launch_norm<__half, __half>(a, vec, st);
    return n->residual_dtype == JQ_F32 ? launch_norm<__nv_bfloat16, float>(a, vec, st) : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
}
