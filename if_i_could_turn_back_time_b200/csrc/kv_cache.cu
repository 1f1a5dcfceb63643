// Writing into the 8-bit key/value cache and reading it back.
#include "kv.cuh"

namespace jqkv {

struct AppendArgs {
    Batch b;
    const void *x[2];                 // keys, values
    long long st[2], sh[2];           // elements between tokens and heads
    uint8_t *codes[2];
    float *scales[2];
    int H, D, touched, vec;
    int most;                         // rows that the shared memory has room for: new tokens of a block
};

// Eight values of a row, as they lie.
template <class T> struct Eight { uint2 w[sizeof(T)]; };
template <class T>
__device__ __forceinline__ Eight<T> load8(const T *p, bool vec) {
    Eight<T> r;
    if (vec) {
        const uint4 *q = reinterpret_cast<const uint4 *>(p);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 u = __ldg(q + i);
            r.w[2 * i] = make_uint2(u.x, u.y);
            r.w[2 * i + 1] = make_uint2(u.z, u.w);
        }
    } else {
        T *e = reinterpret_cast<T *>(&r);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
    return r;
}

// The largest size among them, NaN left out.
__device__ __forceinline__ float largest(const Eight<float> &v) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(__uint_as_float(v.w[i].x)), fabsf(__uint_as_float(v.w[i].y))));
    return m;
}
template <class T, class T2>
__device__ __forceinline__ float largest16(const Eight<T> &v) {
    T2 m = __habs2(*reinterpret_cast<const T2 *>(&v.w[0].x));
    m = __hmax2(m, __habs2(*reinterpret_cast<const T2 *>(&v.w[0].y)));
    m = __hmax2(m, __habs2(*reinterpret_cast<const T2 *>(&v.w[1].x)));
    m = __hmax2(m, __habs2(*reinterpret_cast<const T2 *>(&v.w[1].y)));
    return fmaxf(fmaxf((float)m.x, (float)m.y), 0.f);
}
__device__ __forceinline__ float largest(const Eight<__half> &v) { return largest16<__half, __half2>(v); }
__device__ __forceinline__ float largest(const Eight<__nv_bfloat16> &v) { return largest16<__nv_bfloat16, __nv_bfloat162>(v); }

// The code of x at this scale: the quotient, rounded to fp32 and then to the format's nearest value, ties to even.  Infinities are
// the largest codes, NaN is 0 (a block's one scale cannot hold either).
template <bool E4M3>
__device__ __forceinline__ uint32_t code_of(float q) {
    const float top = E4M3 ? kTopE4m3 : kTopInt8;
    q = q != q ? 0.f : fminf(fmaxf(q, -top), top);
    if (!E4M3) return (uint32_t)(__float2int_rn(q) + 128);
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(q));
    return r & 0xffu;
}
template <bool E4M3>
__device__ __forceinline__ uint32_t encode(float x, float scale) { return code_of<E4M3>(__fdiv_rn(x, scale)); }

// Four codes at once.  The quotient lies between the products with a reciprocal 2^-21 too small and one as much too large, and rounding to
// codes keeps the order: where both have the same code it is the quotient's, elsewhere (one value of 10^4 or fewer, and NaN) the
// quotient is formed.  (Divisions for all values: 48 instructions a value, 69 us for 19184 tokens of 8 x 128 keys and values.)
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float low, float high, float scale) {
    uint32_t r, other;
    if (E4M3) {
        uint16_t a, b, c, d;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(x[1] * low), "f"(x[0] * low));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(x[3] * low), "f"(x[2] * low));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(x[1] * high), "f"(x[0] * high));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(x[3] * high), "f"(x[2] * high));
        r = (uint32_t)a | (uint32_t)b << 16;
        other = r ^ ((uint32_t)c | (uint32_t)d << 16);
        other |= ((r & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;                // NaN's code
    } else {
        uint32_t n[4];
        other = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {                      // 1.5 2^23 + 128 more: the code is the sum's last byte, the others are known
            n[k] = __float_as_uint(fmaf(x[k], low, 12583040.f));
            other |= (n[k] ^ __float_as_uint(fmaf(x[k], high, 12583040.f))) | ((n[k] ^ 0x4b400000u) & 0xffffff00u);
        }
        r = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    }
    if (other) r = encode<E4M3>(x[0], scale) | encode<E4M3>(x[1], scale) << 8 | encode<E4M3>(x[2], scale) << 16 | encode<E4M3>(x[3], scale) << 24;
    return r;
}
template <bool E4M3>
__device__ __forceinline__ float decode(uint32_t code) {
    uint32_t lo, hi;
    codes_to_h4<E4M3>(code, lo, hi);
    return __half2float(__ushort_as_half((unsigned short)(lo & 0xffffu)));
}

// One CTA per block that receives tokens, head, and keys or values.  The new tokens' rows come in once, into shared memory (rows 8 bytes
// longer than they are, so that the lanes that gather a piece of the values meet different banks), with their maximum; then the block's
// scale; then the codes, a 16-byte piece of the cache's order per thread.  19184 tokens of 8 x 128 keys and values, bf16 to e4m3: 53 us, 118 MB moved
// (2.2 TB/s; bound by instructions, most of them the two-byte loads and conversions of the values' pieces).
template <class T, bool E4M3>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs p) {
    extern __shared__ __align__(16) unsigned char rows[];
    __shared__ float red[8];
    const int i = blockIdx.x / p.touched, h = blockIdx.y, what = blockIdx.z, BT = p.b.T, D = p.D;
    int row0;
    const int n = p.b.count(i, row0), len = p.b.length(i);
    const int first = len - n;
    const int blk = (first > 0 ? first >> p.b.shift : 0) + (int)(blockIdx.x % p.touched);
    const int t0 = max(first, blk * BT), t1 = min(min(len, (blk + 1) * BT), t0 + p.most);
    if (n == 0 || t0 >= t1) return;
    const int id = p.b.block(i, t0);                             // (looked at behind the rows, which need not wait for it)
    const T *x = reinterpret_cast<const T *>(p.x[what]) + (long long)(row0 + t0 - first) * p.st[what] + h * p.sh[what];
    const int per = D / 8, pitch = D * (int)sizeof(T) + 8;
    float m = 0.f;
    constexpr int L = sizeof(T) == 2 ? 4 : 2;              // pieces of a thread whose loads are in flight together
    for (int e0 = threadIdx.x; e0 < (t1 - t0) * per; e0 += 256 * L) {
        Eight<T> v[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int e = e0 + 256 * j, r = e / per, c = e - r * per;
            if (e < (t1 - t0) * per) v[j] = load8(x + r * p.st[what] + c * 8, p.vec);
        }
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int e = e0 + 256 * j, r = e / per, c = e - r * per;
            if (e >= (t1 - t0) * per) break;
            uint2 *dst = reinterpret_cast<uint2 *>(rows + r * pitch + c * 8 * sizeof(T));
#pragma unroll
            for (int k = 0; k < (int)sizeof(T); ++k) dst[k] = v[j].w[k];
            m = fmaxf(m, largest(v[j]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
    if (id < 0) return;
    if (m > 3.402823466e38f) {                                   // an infinity among them: the largest of the others
        m = 0.f;
        for (int e = threadIdx.x; e < (t1 - t0) * D; e += 256) {
            const float a = fabsf((float)reinterpret_cast<const T *>(rows + e / D * pitch)[e % D]);
            if (a <= 3.402823466e38f) m = fmaxf(m, a);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
    }
    uint8_t *codes = p.codes[what] + ((size_t)id * p.H + h) * BT * D;
    float *scale_at = p.scales[what] + (size_t)id * p.H + h;
    const int held = t0 - blk * BT, end = t1 - blk * BT;         // places of the block: [0, held) old, [held, end) new
    const float old = held > 0 ? *scale_at : 0.f;
    const float scale = fmaxf(old, __fdiv_rn(fmaxf(m, kLeastMax), E4M3 ? kTopE4m3 : kTopInt8));
    const float inv = 1.f / scale, low = inv - inv * 4.76837158e-7f, high = inv + inv * 4.76837158e-7f;       // 2^-21
    const bool grown = held > 0 && scale > old;
    __syncthreads();
    if (threadIdx.x == 0) *scale_at = scale;
    const int g0 = (grown ? 0 : held) / 16, g1 = (end + 15) / 16;
    for (int e = threadIdx.x + g0 * D; e < g1 * D; e += 256) {                // pieces of 16 bytes, D of them in a group of 16 tokens
        const int group = e / D, c = (e - group * D) >> 5, g = e % 32 / 4, t = e % 4;
        uint4 *at = reinterpret_cast<uint4 *>(codes) + e;
        // (a piece of new tokens alone is not read)
        uint4 w = group * 16 >= held && group * 16 + 16 <= end ? make_uint4(0, 0, 0, 0) : *at;
        uint32_t *word = &w.x;
        if (what == 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int token = group * 16 + 4 * (g >> 1) + (g & 1) + 2 * j;
                if (token >= held && token < end) {
                    const T *v = reinterpret_cast<const T *>(rows + (token - held) * pitch) + c * 32 + t * 8;
                    Eight<T> u;
#pragma unroll
                    for (int k = 0; k < (int)sizeof(T); ++k) u.w[k] = reinterpret_cast<const uint2 *>(v)[k];
                    const T *f = reinterpret_cast<const T *>(&u);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float x4[4] = {(float)f[4 * k], (float)f[4 * k + 1], (float)f[4 * k + 2], (float)f[4 * k + 3]};
                        word[2 * j + k] = encode4<E4M3>(x4, low, high, scale);
                    }
                } else if (grown && token < held) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t x4 = 0;
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            x4 |= encode<E4M3>(__fmul_rn(decode<E4M3>(word[2 * j + k] >> 8 * b & 255), old), scale) << 8 * b;
                        word[2 * j + k] = x4;
                    }
                }
            }
        } else {
            const int token0 = group * 16 + 4 * t;
            if (token0 >= held && token0 + 4 <= end) {
                const T *row = reinterpret_cast<const T *>(rows + (token0 - held) * pitch) + c * 32 + g;
                const int next = pitch / (int)sizeof(T);
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const float x4[4] = {(float)row[dt * 8], (float)row[next + dt * 8], (float)row[2 * next + dt * 8], (float)row[3 * next + dt * 8]};
                    word[dt] = encode4<E4M3>(x4, low, high, scale);
                }
            } else {
#pragma unroll 1
                for (int b = 0; b < 4; ++b) {
                    const int token = token0 + b;
                    const bool fresh = token >= held && token < end;
                    if (!fresh && !(grown && token < held)) continue;
                    const T *row = reinterpret_cast<const T *>(rows + (token - held) * pitch) + c * 32 + g;
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt) {
                        const uint32_t was = word[dt] >> 8 * b & 255;
                        const uint32_t is = encode<E4M3>(fresh ? (float)row[dt * 8] : __fmul_rn(decode<E4M3>(was), old), scale);
                        word[dt] ^= (was ^ is) << 8 * b;
                    }
                }
            }
        }
        *at = w;
    }
}

struct ReadArgs {
    Batch b;
    const uint8_t *codes[2];
    const float *scales[2];
    void *out[2];
    int H, D, last, groups, dtype;
};

// A warp per group of 16 tokens and head: what the codes stand for, in the order of a user's tensors.  The last 4159 tokens of eight sequences,
// fp32: 63 us, 310 MB (4.9 TB/s), nearly all of it writing.
template <bool E4M3>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadArgs p) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int h = (int)(job % p.H), what = blockIdx.y;
    const long long k = job / p.H;
    const int i = (int)(k / p.groups);
    if (i >= p.b.S) return;
    const int begin = p.b.length(i) - p.last;                                 // (below 0: places before the first token read as 0)
    const int group = (begin >= 0 ? begin / 16 : -((15 - begin) / 16)) + (int)(k % p.groups);
    const int base = group * 16 - begin;                                      // place of the group's first token in the output
    if (base >= p.last) return;
    const int id = group >= 0 ? p.b.block(i, group * 16) : -1;
    const float scale = id >= 0 ? p.scales[what][(size_t)id * p.H + h] : 0.f;
    const uint4 *at = reinterpret_cast<const uint4 *>(p.codes[what] + (((size_t)max(id, 0) * p.H + h) * p.b.T + (group >= 0 ? group * 16 & (p.b.T - 1) : 0)) * p.D);
    const size_t row = (size_t)p.H * p.D;
    const size_t out0 = (size_t)i * p.last * row + (size_t)h * p.D;
    for (int c = 0; c < p.D / 32; ++c) {
        const uint4 w = id >= 0 ? at[c * 32 + lane] : make_uint4(0, 0, 0, 0);
        const uint32_t word[4] = {w.x, w.y, w.z, w.w};
        float v[16];
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
            uint32_t lo, hi;
            codes_to_h4<E4M3>(word[k4], lo, hi);
            const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
            v[4 * k4] = a.x; v[4 * k4 + 1] = a.y; v[4 * k4 + 2] = b.x; v[4 * k4 + 3] = b.y;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = id >= 0 ? __fmul_rn(v[e], scale) : 0.f;
        if (what == 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int place = base + 4 * (g >> 1) + (g & 1) + 2 * j;
                if (place < 0 || place >= p.last) continue;
                const size_t o = out0 + place * row + c * 32 + t * 8;
                if (p.dtype == JQ_F32) {
                    float4 *q = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.out[0]) + o);
                    q[0] = make_float4(v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3]);
                    q[1] = make_float4(v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) jq::store_out(p.out[0], o + e, v[8 * j + e], p.dtype);
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int place = base + 4 * t + b;
                if (place < 0 || place >= p.last) continue;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) jq::store_out(p.out[1], out0 + place * row + c * 32 + dt * 8 + g, v[4 * dt + b], p.dtype);
            }
        }
    }
}

// What every entry asks of a cache and its sequences; JQ_OK or the refusal.
int check_cache(const jq_kv_cache *c, const jq_kv_batch *s) {
    if (!c || !s || !c->keys || !c->values || !c->key_scales || !c->value_scales) return JQ_ERR_NULL_PTR;
    if (s->sequences != 0 && (!s->table || !s->lengths)) return JQ_ERR_NULL_PTR;
    if (c->fmt != JQ_KV_INT8 && c->fmt != JQ_KV_E4M3) return JQ_ERR_BAD_DTYPE;
    if (c->blocks <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535 || c->head_dim <= 0 || c->head_dim % 32 || c->head_dim > 256 ||
        (c->block_size != 16 && c->block_size != 32 && c->block_size != 64 && c->block_size != 128))
        return JQ_ERR_BAD_SHAPE;
    if (s->sequences < 0 || s->table_width <= 0 || s->table_stride < s->table_width || s->tokens < 0 ||
        (long long)s->table_width * c->block_size > 0x7fffff00LL)
        return JQ_ERR_BAD_SHAPE;
    if (s->sequences ? !s->starts && s->tokens % s->sequences : s->tokens) return JQ_ERR_BAD_SHAPE;
    if (!jq_aligned16(c->keys) || !jq_aligned16(c->values) || (reinterpret_cast<uintptr_t>(c->key_scales) & 3u) ||
        (reinterpret_cast<uintptr_t>(c->value_scales) & 3u) || (reinterpret_cast<uintptr_t>(s->table) & 3u) ||
        (reinterpret_cast<uintptr_t>(s->lengths) & 3u) || (reinterpret_cast<uintptr_t>(s->starts) & 3u))
        return JQ_ERR_BAD_ALIGN;
    return JQ_OK;
}

Batch batch_of(const jq_kv_cache *c, const jq_kv_batch *s) {
    Batch b{};
    b.table = s->table; b.lengths = s->lengths; b.starts = s->starts;
    b.S = s->sequences; b.width = s->table_width; b.table_stride = s->table_stride; b.tokens = s->tokens;
    b.each = s->sequences ? s->tokens / s->sequences : 0;
    b.T = c->block_size; b.blocks = c->blocks;
    while (1 << b.shift < b.T) ++b.shift;
    return b;
}

// Most new tokens of a sequence: what the caller says, at most all of them.
int most_new(const jq_kv_batch *s) {
    if (!s->starts) return s->sequences ? s->tokens / s->sequences : 0;
    return s->max_new > 0 && s->max_new < s->tokens ? s->max_new : s->tokens;
}

}  // namespace jqkv

using namespace jqkv;

extern "C" int jq_kv_append(const jq_kv_cache *c, const jq_kv_batch *s, const void *k, const void *v, const int64_t *stride_k,
                            const int64_t *stride_v, int dtype, jq_stream_t stream) {
    const int bad = check_cache(c, s);
    if (bad) return bad;
    if (dtype < 0 || dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (s->sequences == 0 || s->tokens == 0) return JQ_OK;
    if (!k || !v || !stride_k || !stride_v) return JQ_ERR_NULL_PTR;
    const unsigned esz = dtype == JQ_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & (esz - 1)) return JQ_ERR_BAD_ALIGN;
    AppendArgs a{};
    a.b = batch_of(c, s);
    a.x[0] = k; a.x[1] = v;
    a.st[0] = stride_k[0]; a.sh[0] = stride_k[1]; a.st[1] = stride_v[0]; a.sh[1] = stride_v[1];
    a.codes[0] = reinterpret_cast<uint8_t *>(c->keys); a.codes[1] = reinterpret_cast<uint8_t *>(c->values);
    a.scales[0] = c->key_scales; a.scales[1] = c->value_scales;
    a.H = c->kv_heads; a.D = c->head_dim;
    const long long most = most_new(s);
    a.touched = (int)((most + c->block_size - 2) / c->block_size + 1);
    if (a.touched > s->table_width) a.touched = s->table_width;
    const long long piece = 16 / esz;
    a.vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 &&
            (a.st[0] | a.sh[0] | a.st[1] | a.sh[1]) % piece == 0;
    const long long grid = (long long)a.touched * s->sequences;
    if (grid > 0x7fffffffLL) return JQ_ERR_BAD_SHAPE;
    const dim3 blocks((unsigned)grid, (unsigned)c->kv_heads, 2);
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    void (*const kernels[3][2])(const AppendArgs) = {{append_kernel<float, false>, append_kernel<float, true>},
                                                     {append_kernel<__half, false>, append_kernel<__half, true>},
                                                     {append_kernel<__nv_bfloat16, false>, append_kernel<__nv_bfloat16, true>}};
    const bool e = c->fmt == JQ_KV_E4M3;
    static jq_contexts done[3][2];
    a.most = most < c->block_size ? (int)most : c->block_size;
    const int bytes = a.most * (c->head_dim * (int)esz + 8);
    JQ_CUDA_TRY(jq_allow_smem(reinterpret_cast<const void *>(kernels[dtype][e]), 128 * (256 * (int)esz + 8), done[dtype][e]));
    kernels[dtype][e]<<<blocks, 256, bytes, st>>>(a);
    return jq_launch_status();
}

extern "C" int jq_kv_read(const jq_kv_cache *c, const jq_kv_batch *s, int last, void *k, void *v, int dtype, jq_stream_t stream) {
    const int bad = check_cache(c, s);
    if (bad) return bad;
    if (dtype < 0 || dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (last < 0) return JQ_ERR_BAD_SHAPE;
    if (s->sequences == 0 || last == 0) return JQ_OK;
    if (!k || !v) return JQ_ERR_NULL_PTR;
    if (!jq_aligned16(k) || !jq_aligned16(v)) return JQ_ERR_BAD_ALIGN;
    ReadArgs a{};
    a.b = batch_of(c, s);
    a.codes[0] = reinterpret_cast<const uint8_t *>(c->keys); a.codes[1] = reinterpret_cast<const uint8_t *>(c->values);
    a.scales[0] = c->key_scales; a.scales[1] = c->value_scales;
    a.out[0] = k; a.out[1] = v;
    a.H = c->kv_heads; a.D = c->head_dim; a.last = last; a.groups = last / 16 + 2; a.dtype = dtype;
    const long long jobs = (long long)a.groups * s->sequences * c->kv_heads, grid = (jobs + 7) / 8;
    if (grid > 0x7fffffffLL) return JQ_ERR_BAD_SHAPE;
    (c->fmt == JQ_KV_E4M3 ? read_kernel<true> : read_kernel<false>)<<<dim3((unsigned)grid, 2), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    return jq_launch_status();
}
