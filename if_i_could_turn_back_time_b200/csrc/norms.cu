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
    int layer, post, rotate;
    int wdtype, gdtype;                // types of the four vectors and of the gate
    int wide_w, wide_g;                // fp32 rather than of x's type
};

// Eight values of a vector of T or of fp32 (weights, gates).  The piece that is enough for T is asked for ahead of its use (a gate's
// with the row: 197 x 256 rows of 768 fp16, gated by image, 72 us without and 63 with; weights, which the caches have, behind the sums: asked for
// ahead of them they cost registers, 8191 x 4096 bf16 45 us against 43); the second one of fp32 at its use.
template <class T> struct Piece {
    uint4 a;
    __device__ __forceinline__ static const uint4 *at(const void *p, bool wide, int i) {
        return reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned char *>(p) + (size_t)i * (wide ? 4 : sizeof(T)));
    }
    __device__ __forceinline__ void ask(const void *p, bool wide, int i, int width) { a = i < width ? *at(p, wide, i) : make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(const void *p, bool wide, int i, int width, float (&v)[8]) const {
        if (sizeof(T) == 4 || wide) {
            Raw8<float> r;
            r.w[0] = a;
            r.w[1] = i < width ? at(p, true, i)[1] : make_uint4(0, 0, 0, 0);
            widen(r, v);
        } else if constexpr (sizeof(T) == 2) {
            Raw8<T> r;
            r.w[0] = a;
            widen(r, v);
        }
    }
};

// Blocks that an SM is to hold: more of them hide more of a row's chain of loads and sums, as long as what no longer fits in registers stays little.
// us at 3 / 4 / unbounded (2 or 3): 50432 x 768 fp16, three chunks a thread - / 54 / 63; bf16 with an fp32 stream 74 / - / 80; 50000 x 500, two chunks
// - / 37 / 48; 20000 x 1024, four chunks: bf16 with its stream of 16 bits 46 at 4 and 34 unbounded, of 32 bits 47 at 3 and 43, fp32 56 at 3 and 59.
// Blocks of 256 threads, 8191 x 4096 with both norms and an fp32 stream, calls one behind another on inputs that take turns: 74 at 4, 78 at 5, 79 unbounded.
constexpr int resident(int threads, int chunks, int x_size, int r_size) {
    if (threads) return threads == 256 ? 4 : 1;
    if (chunks < 3) return 4;
    if (chunks == 3) return r_size == 2 ? 4 : 3;
    return x_size == 4 || r_size == 2 ? 3 : 1;
}

// A warp (kThreads 0) or a block per row, which stays in registers from the first read to the last write:
//   u = N(x) post_weight + post_bias (or x),  r = residual + scale * (gate * u),  h = N(r) weight + bias,
// N(v) = v / sqrt(mean(v^2) + eps), or of v - mean(v).  All in fp32; h follows from r as it was before its rounding.
// Bound by memory: 8191 x 4096 with both norms and an fp32 stream 68 us in a graph (5.9 TB/s), 70 to 74 in calls one behind another; with codes in
// place of h 72, rotated 79; one norm in bf16 44, 47 and 56 (codes: 5.0 and 4.2 TB/s; the rotation has four shuffles a value here).  50432 x 768
// fp16 with a gate for each image 54 (5.8), 50000 x 197 23, 4000 x 5025 44 (3.6: one-element loads).  Two chunks a thread and code without paths that a call does not take are what did it (four chunks,
// every alignment and type in one kernel: 104, 72, 69 and 79; instructions waited for the instruction cache).
// kPieces: every row and vector is of 16-byte pieces, and vectors are of T or fp32; kPairs: rows are of pairs; kScattered: any width, alignment,
// stride and type.
template <class T, class R, int kChunks, int kThreads, Lay L>
__global__ void __launch_bounds__(kThreads ? kThreads : 256, resident(kThreads, kChunks, sizeof(T), sizeof(R))) norm_kernel(const __grid_constant__ NormArgs p) {
    constexpr bool kBlock = kThreads != 0;
    __shared__ Shared sh;
    jqta::pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int threads = kBlock ? blockDim.x : 32, me = kBlock ? threadIdx.x : lane;
    const int row = kBlock ? blockIdx.x : blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.stride_x;
    const auto first = [&](int j) { return first_of<L>(me + j * threads); };
    Joined<kBlock> joined(sh);
    const float each = 1.f / (float)p.width;
    float v[kChunks][8];
    Held<L, R> res[kChunks];
    Piece<T> gates[kChunks];
    const unsigned char *gate = reinterpret_cast<const unsigned char *>(p.gate);
    if (gate) gate += ((row / p.inner) * p.gate_outer + (row % p.inner) * p.gate_inner) * (p.gdtype == JQ_F32 ? 4 : 2);
    {
        Held<L, T> held[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) held[j].load(x, first(j), p.width);
        if (p.residual) {
            const R *from = reinterpret_cast<const R *>(p.residual) + row * p.stride_res;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) res[j].load(from, first(j), p.width);
        }
        if (L == kPieces && gate && !p.gate_one) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) gates[j].ask(gate, p.wide_g, first(j), p.width);
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j) held[j].get(v[j]);
    }
    // whether element k of chunk j is one of the row
    auto in = [&](int j, int k) { return inside<L>(first(j), k, p.width); };
    auto normed = [&](const void *weight, const void *bias) {
        Piece<T> piece[kChunks];
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
            if (L == kPieces) {
#pragma unroll
                for (int j = 0; j < kChunks; ++j) piece[j].ask(weight, p.wide_w, first(j), p.width);
            }
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float w[8];
                if constexpr (L == kPieces) piece[j].get(weight, p.wide_w, first(j), p.width, w);
                else load_any<L>(weight, p.wdtype, first(j), p.width, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= w[k];
            }
        }
        if (bias) {
            if (L == kPieces) {
#pragma unroll
                for (int j = 0; j < kChunks; ++j) piece[j].ask(bias, p.wide_w, first(j), p.width);
            }
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float b[8];
                if constexpr (L == kPieces) piece[j].get(bias, p.wide_w, first(j), p.width, b);
                else load_any<L>(bias, p.wdtype, first(j), p.width, b);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] += b[k];
            }
        }
    };
    if (p.post) normed(p.post_weight, p.post_bias);
    float f = p.scale;
    if (gate) {
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
                if constexpr (L == kPieces) gates[j].get(gate, p.wide_g, first(j), p.width, g);
                else load_any<L>(gate, p.gdtype, first(j), p.width, g);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= g[k];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        if (p.residual) {
            float old[8];
            res[j].get(old);
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
        for (int j = 0; j < kChunks; ++j) store_chunk<L>(r, first(j), p.width, v[j]);
    }
    // (an infinite gate or root times the zeros behind the row's end is NaN)
    if (p.post || gate) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] = in(j, k) ? v[j][k] : 0.f;
    }
    normed(p.weight, p.bias);
    if (!p.codes) {
        T *h = reinterpret_cast<T *>(p.h) + (long long)row * p.width;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) store_chunk<L>(h, first(j), p.width, v[j]);
        return;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        if (L == kPieces && p.rotate) {
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
    for (int j = 0; j < kChunks; ++j) coder.template store_as<L>(codes, first(j), p.width, v[j]);
}

// ---- host side -------------------------------------------------------------------------

template <class T, class R>
static int launch_norm(const NormArgs &a, Lay l, cudaStream_t st) {
    const int chunks = chunks_of(a.width, l);
    Cut c = cut_of(chunks, a.rows, jq_sm_count(), 2);
    // (rows by elements: four chunks of a warp's thread are some hundred registers, and a block of two warps is ahead)
    if (l != kPieces && c.threads == 0 && c.chunks > 2) c = Cut{2, (chunks / 2 + 31) / 32 * 32};
    void (*k)(const NormArgs);
    if (l == kPieces) {
        if (c.threads == 0) k = c.chunks == 1 ? norm_kernel<T, R, 1, 0, kPieces> : c.chunks == 2 ? norm_kernel<T, R, 2, 0, kPieces> :
                                c.chunks == 3 ? norm_kernel<T, R, 3, 0, kPieces> : norm_kernel<T, R, 4, 0, kPieces>;
        else k = c.chunks == 1 ? norm_kernel<T, R, 1, 1024, kPieces> : c.chunks == 2 ? (c.threads <= 256 ? norm_kernel<T, R, 2, 256, kPieces> : norm_kernel<T, R, 2, 1024, kPieces>) : norm_kernel<T, R, 4, 1024, kPieces>;
    } else if (l == kPairs) {
        if (c.threads == 0) k = c.chunks == 1 ? norm_kernel<T, R, 1, 0, kPairs> : norm_kernel<T, R, 2, 0, kPairs>;
        else k = c.chunks <= 2 ? norm_kernel<T, R, 2, 1024, kPairs> : norm_kernel<T, R, 4, 1024, kPairs>;
    } else {
        if (c.threads == 0) k = c.chunks == 1 ? norm_kernel<T, R, 1, 0, kScattered> : norm_kernel<T, R, 2, 0, kScattered>;
        else k = c.chunks <= 2 ? norm_kernel<T, R, 2, 1024, kScattered> : norm_kernel<T, R, 4, 1024, kScattered>;
    }
    k<<<c.threads ? a.rows : (a.rows + 7) / 8, c.threads ? c.threads : 256, 0, st>>>(a);
    return jq_launch_status();
}

}  // namespace jq8

using namespace jq8;

extern "C" int jq_residual_norm(const jq_norm *n, jq_stream_t stream) {
    if (!n || !n->x || (!n->h && !n->codes) || (n->codes && !n->scales)) return JQ_ERR_NULL_PTR;
    if (n->rows <= 0 || n->rows > JQ_INT8_MAX_ROWS || n->width <= 0 || n->width > kMostKept || n->stride_x < 0 || n->stride_residual < 0) return JQ_ERR_BAD_SHAPE;
    if (n->kind != JQ_NORM_RMS && n->kind != JQ_NORM_LAYER) return JQ_ERR_UNSUPPORTED;
    if (n->had_block != 0 && (n->had_block != 128 || n->width % 128 || !n->codes)) return JQ_ERR_BAD_SHAPE;
    if (n->gate && n->gate_inner_rows <= 0) return JQ_ERR_BAD_SHAPE;
    const int types[4] = {n->x_dtype, n->residual_dtype, n->weight_dtype, n->gate_dtype};
    for (int t : types)
        if (t < 0 || t > 2) return JQ_ERR_BAD_DTYPE;
    if (n->residual_dtype != n->x_dtype && n->residual_dtype != JQ_F32) return JQ_ERR_BAD_DTYPE;
    if (n->codes && (!jq_aligned16(n->codes) || n->stride_codes % 16)) return JQ_ERR_BAD_ALIGN;
    if (n->codes && n->stride_codes < n->width) return JQ_ERR_BAD_SHAPE;
    if (n->reserved) return JQ_ERR_BAD_SHAPE;
    const int W = n->width, xs = n->x_dtype == JQ_F32 ? 4 : 2, rs = n->residual_dtype == JQ_F32 ? 4 : 2;
    const int ws = n->weight_dtype == JQ_F32 ? 4 : 2, gs = n->gate_dtype == JQ_F32 ? 4 : 2;
    if (!jq_whole(n->x, xs) || !jq_whole(n->h, xs) || !jq_whole(n->residual, rs) || !jq_whole(n->r, rs) || !jq_whole(n->weight, ws) || !jq_whole(n->bias, ws) ||
        !jq_whole(n->post_weight, ws) || !jq_whole(n->post_bias, ws) || !jq_whole(n->gate, gs) || (n->codes && !jq_whole(n->scales, 4)))
        return JQ_ERR_BAD_ALIGN;
    NormArgs a{};
    a.x = n->x; a.residual = n->residual; a.r = n->r; a.h = n->h; a.codes = reinterpret_cast<int8_t *>(n->codes); a.scales = n->scales;
    a.weight = n->weight; a.bias = n->bias; a.post_weight = n->post_weight; a.post_bias = n->post_bias; a.gate = n->gate;
    a.stride_x = n->stride_x; a.stride_res = n->stride_residual; a.stride_q = n->stride_codes;
    a.gate_outer = n->gate_outer; a.gate_inner = n->gate_inner; a.inner = n->gate ? n->gate_inner_rows : 1; a.gate_one = n->gate_one;
    a.rows = n->rows; a.width = W; a.scale = n->scale; a.eps = n->eps;
    a.layer = n->kind == JQ_NORM_LAYER; a.post = n->post; a.rotate = n->had_block != 0;
    a.wdtype = n->weight_dtype; a.gdtype = n->gate_dtype;
    a.wide_w = n->weight_dtype == JQ_F32;
    a.wide_g = n->gate_dtype == JQ_F32;
    const bool vectors = n->weight || n->bias || n->post_weight || n->post_bias;
    const bool vec = W % 8 == 0 && aligned(n->x, n->stride_x, xs) && aligned(n->residual, n->stride_residual, rs) && jq_aligned16(n->r) && jq_aligned16(n->h) &&
                     jq_aligned16(n->weight) && jq_aligned16(n->bias) && jq_aligned16(n->post_weight) && jq_aligned16(n->post_bias) &&
                     (!vectors || n->weight_dtype == n->x_dtype || a.wide_w) &&
                     (!n->gate || n->gate_one || (aligned(n->gate, n->gate_outer, gs) && n->gate_inner * gs % 16 == 0 && (n->gate_dtype == n->x_dtype || a.wide_g)));
    if (a.rotate && !vec) return JQ_ERR_BAD_ALIGN;
    auto paired = [](const void *p, int64_t stride, int size) { return (reinterpret_cast<uintptr_t>(p) & (2 * size - 1)) == 0 && stride % 2 == 0; };
    const bool pairs = W % 2 == 0 && paired(n->x, n->stride_x, xs) && paired(n->residual, n->stride_residual, rs) && paired(n->r, 0, rs) && paired(n->h, 0, xs);
    const Lay lay = vec ? kPieces : pairs ? kPairs : kScattered;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (n->x_dtype == JQ_F32) return launch_norm<float, float>(a, lay, st);
    if (n->x_dtype == JQ_F16) return n->residual_dtype == JQ_F32 ? launch_norm<__half, float>(a, lay, st) : launch_norm<__half, __half>(a, lay, st);
    return n->residual_dtype == JQ_F32 ? launch_norm<__nv_bfloat16, float>(a, lay, st) : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, lay, st);
}
