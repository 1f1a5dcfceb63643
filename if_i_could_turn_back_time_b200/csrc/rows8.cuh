// Rows of activations in 8-bit integers: what the kernels that write them share (sm_100a).
//
// A row x (K values) has one fp32 scale s = max(|x|, 2^-100) / 127 and the codes q = x / s, the fp32 quotient rounded to the nearest
// integer, ties to even: -127 .. 127, and 0 stays 0.  A row with a NaN or an infinity has the scale NaN and codes 0, so that every
// product of it is NaN, as it would be without codes.  Rows of codes lie a multiple of 16 bytes apart.
#pragma once
#include "tc.cuh"

namespace jq8 {

constexpr float kLeastMax = 7.888609052210118e-31f;   // 2^-100: the least maximum that a scale is made of, so that its reciprocal is finite
constexpr uint32_t kInf = 0x7f800000u;

template <class T> struct Raw8 { uint4 w[sizeof(T) / 2]; };          // eight values as they lie

__device__ __forceinline__ void widen(const Raw8<float> &r, float (&v)[8]) {
    const uint32_t *u = &r.w[0].x, *w = &r.w[1].x;
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(u[i]); v[4 + i] = __uint_as_float(w[i]); }
}
__device__ __forceinline__ void widen(const Raw8<__half> &r, float (&v)[8]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&r.w[0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}
__device__ __forceinline__ void widen(const Raw8<__nv_bfloat16> &r, float (&v)[8]) {
    const uint32_t *u = &r.w[0].x;
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}

// Which elements of a row chunk c holds.  Rows whose width is a multiple of 8: eight neighbours.  Others: eight that are 32 apart, so
// that a warp's one-element loads and stores lie side by side.
struct Places {
    int width, next;                   // next: between a chunk's elements
    __device__ __forceinline__ Places(int width, bool neighbours) : width(width), next(neighbours ? 1 : 32) {}
    __device__ __forceinline__ int first(int c) const { return next == 1 ? c * 8 : (c >> 5) * 256 + (c & 31); }
};

// A chunk of a row; zeros behind its end.  vec: the row is 16-byte aligned and its chunks are neighbours.
template <class T>
__device__ __forceinline__ Raw8<T> load_chunk(const T *row, int c, const Places &at, bool vec) {
    Raw8<T> r;
    const int i = at.first(c);
    if (vec) {
        const bool in = i < at.width;
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k)
            r.w[k] = in ? *reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned char *>(row + i) + 16 * k) : make_uint4(0, 0, 0, 0);
    } else {
        T *e = reinterpret_cast<T *>(&r);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = i + k * at.next < at.width ? row[i + k * at.next] : (T)0.f;
    }
    return r;
}
template <class T>
__device__ __forceinline__ void store_chunk(T *row, int c, const Places &at, bool vec, const float (&v)[8]) {
    const int i = at.first(c);
    if (vec) {
        if (i >= at.width) return;
        Raw8<T> r;
        T *e = reinterpret_cast<T *>(&r);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = (T)v[k];
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) *reinterpret_cast<uint4 *>(reinterpret_cast<unsigned char *>(row + i) + 16 * k) = r.w[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k * at.next < at.width) row[i + k * at.next] = (T)v[k];
    }
}
// The same from a vector of any of the three types (weights: the same for every row, so that they come from the caches).
__device__ __forceinline__ void load_any(const void *row, int dtype, int c, const Places &at, bool vec, float (&v)[8]) {
    if (dtype == JQ_BF16) widen(load_chunk(reinterpret_cast<const __nv_bfloat16 *>(row), c, at, vec), v);
    else if (dtype == JQ_F16) widen(load_chunk(reinterpret_cast<const __half *>(row), c, at, vec), v);
    else widen(load_chunk(reinterpret_cast<const float *>(row), c, at, vec), v);
}

// Rotation of 128 neighbours: 16 / A lanes with 8 A of them each, in the order of stages (strides 1, 2, .., 64; sums in the lower place,
// differences in the upper) of fwht128_warp, so that both give the same bits.  Between lanes a stage is one shuffle and one fused
// multiply-add with 1 or -1, which rounds as the sum or the difference does.  The shuffles bound it: four per value at A = 1, two at A = 4.
template <int A>
__device__ __forceinline__ void rotate128(float (&v)[A][8], int lane) {
#pragma unroll
    for (int m = 1; m < 8 * A; m <<= 1)
#pragma unroll
        for (int j = 0; j < 8 * A; ++j)
            if (!(j & m)) {
                const float a = v[j >> 3][j & 7], b = v[(j | m) >> 3][(j | m) & 7];
                v[j >> 3][j & 7] = a + b;
                v[(j | m) >> 3][(j | m) & 7] = a - b;
            }
#pragma unroll
    for (int m = 1; m < 16 / A; m <<= 1) {
        const float sign = (lane & m) ? -1.f : 1.f;
#pragma unroll
        for (int j = 0; j < 8 * A; ++j) v[j >> 3][j & 7] = fmaf(v[j >> 3][j & 7], sign, __shfl_xor_sync(0xffffffffu, v[j >> 3][j & 7], m));
    }
#pragma unroll
    for (int j = 0; j < 8 * A; ++j) v[j >> 3][j & 7] *= 0.08838834764831845f;
}

// Bits of the largest |v|; NaN is above infinity.
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}
// The same of values as they lie
__device__ __forceinline__ uint32_t largest_bits(const Raw8<float> &r) {
    const uint32_t *u = &r.w[0].x, *w = &r.w[1].x;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, max(u[j] & 0x7fffffffu, w[j] & 0x7fffffffu));
    return m;
}
template <class T>
__device__ __forceinline__ uint32_t largest_pair(const Raw8<T> &r) {                     // two largest sizes, as bits of 16
    const uint4 &w = r.w[0];
    return __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t bits_of_pair(uint32_t m, __nv_bfloat16) { return max(m & 0xffffu, m >> 16) << 16; }
__device__ __forceinline__ uint32_t bits_of_pair(uint32_t m, __half) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16)))) & 0x7fffffffu;
}

// What turns values into codes.  The quotient lies between the products with a reciprocal 2^-21 too small and one as much too large,
// and rounding keeps the order: where both round to one integer it is the quotient's, elsewhere (a value in some 10^4) the quotient
// is formed.  1.5 2^23 more than a product: the sum's last byte is the code.
struct Coder {
    float scale, low, high;
    bool good;
    __device__ __forceinline__ explicit Coder(uint32_t bits) {
        good = bits < kInf;
        scale = __fdiv_rn(fmaxf(__uint_as_float(good ? bits : 0u), kLeastMax), 127.f);
        const float inv = __fdiv_rn(1.f, scale);
        low = inv - inv * 4.76837158e-7f;
        high = inv + inv * 4.76837158e-7f;
    }
    __device__ __forceinline__ float told() const { return good ? scale : __uint_as_float(0x7fffffffu); }
    __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) const {
        const float x[4] = {a, b, c, d};
        uint32_t n[4], other = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            n[k] = __float_as_uint(fmaf(x[k], low, 12582912.f));
            other |= n[k] ^ __float_as_uint(fmaf(x[k], high, 12582912.f));
        }
        if (other) {
#pragma unroll
            for (int k = 0; k < 4; ++k) n[k] = (uint32_t)min(127, max(-127, __float2int_rn(__fdiv_rn(x[k], scale))));
        }
        const uint32_t r = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
        return good ? r : 0u;
    }
    __device__ __forceinline__ uint2 eight(const float (&v)[8]) const { return make_uint2(four(v[0], v[1], v[2], v[3]), four(v[4], v[5], v[6], v[7])); }
    __device__ __forceinline__ void store(int8_t *row, int c, const Places &at, const float (&v)[8]) const {
        const int i = at.first(c);
        const uint2 q = eight(v);
        if (at.next == 1) {
            if (i < at.width) *reinterpret_cast<uint2 *>(row + i) = q;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k * 32 < at.width) row[i + k * 32] = (int8_t)((k < 4 ? q.x : q.y) >> 8 * (k & 3));
        }
    }
};

// Sums and maxima over the threads of a row: a warp, or a block.  The block's forms alternate between two sets of places, so that one
// barrier for each suffices.
struct Shared { float f[2][32]; };
template <bool kBlock> struct Joined {
    Shared &sh;
    int turn = 0;
    __device__ __forceinline__ explicit Joined(Shared &s) : sh(s) {}
    __device__ __forceinline__ float sum(float v) {
        v = jq::warp_sum(v);
        if (!kBlock) return v;
        float *f = sh.f[turn ^= 1];
        if ((threadIdx.x & 31) == 0) f[threadIdx.x >> 5] = v;
        __syncthreads();
        return jq::warp_sum((threadIdx.x & 31) < (blockDim.x >> 5) ? f[threadIdx.x & 31] : 0.f);
    }
    __device__ __forceinline__ uint32_t top(uint32_t v) {
        v = __reduce_max_sync(0xffffffffu, v);
        if (!kBlock) return v;
        uint32_t *f = reinterpret_cast<uint32_t *>(sh.f[turn ^= 1]);
        if ((threadIdx.x & 31) == 0) f[threadIdx.x >> 5] = v;
        __syncthreads();
        return __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < (blockDim.x >> 5) ? f[threadIdx.x & 31] : 0u);
    }
};

// ---- host side

constexpr int kMostKept = 32768;       // longest row that a block keeps in registers: 1024 threads with four chunks of eight values

struct Cut { int chunks, threads; };   // threads 0: a warp per row

// A row's chunks over threads.  Up to 128 chunks a warp has them all and needs no barrier; longer rows have a block, with `many` chunks
// per thread (loads in flight together, few warps at the barriers) unless rows are so few that latency counts: then one.
inline Cut cut_of(int width, bool neighbours, int rows, int sms, int many) {
    const int chunks = neighbours ? (width + 7) / 8 : (width + 255) / 256 * 32;
    if (chunks <= 128 && (rows > 2 * sms || chunks <= 32)) return Cut{(chunks + 31) / 32, 0};
    const int per = chunks > 2048 ? 4 : rows > 2 * sms || chunks > 1024 ? many : 1;
    const int threads = ((chunks + per - 1) / per + 31) / 32 * 32;
    return Cut{per, threads < 1024 ? threads : 1024};
}

inline bool aligned(const void *p, long long stride, int size) {
    return jq_aligned16(p) && stride * size % 16 == 0;
}

}  // namespace jq8
