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

// A chunk is eight elements of a row, whose first one first_of() tells:
//   kPieces     rows of 16-byte pieces: chunk c from 8 c on;
//   kPairs      four pairs of neighbours 64 apart, so that a warp's two-element loads and stores lie side by side: rows of even length and place;
//   kScattered  eight elements 32 apart: whatever else there is.
// (For norms of rows that begin anywhere, chunks that are 16-byte pieces of memory, with a row's first and last one by elements, were slower up
// to some thousand elements: 50000 x 197 bf16 30 us against 24.)
enum Lay { kPieces, kPairs, kScattered };
template <Lay L> __device__ __forceinline__ int first_of(int c) { return L == kPieces ? c * 8 : (c >> 5) * 256 + (L == kPairs ? 2 : 1) * (c & 31); }
template <Lay L> __device__ __forceinline__ constexpr int place(int k) { return L == kPieces ? k : L == kPairs ? (k >> 1) * 64 + (k & 1) : k * 32; }
// whether all of a chunk is the row's (the same for a warp's lanes where they lie side by side), and whether element k is
template <Lay L> __device__ __forceinline__ bool whole(int i, int width) { return L == kPieces ? i < width : (i | 255) < width; }
template <Lay L> __device__ __forceinline__ bool inside(int i, int k, int width) { return L == kPieces ? i < width : i + place<L>(k) < width; }

template <class T> struct alignas(2 * sizeof(T)) PairOf { T a, b; };

// A chunk between its load and its first use, zeros outside the row: as it lies, or, where it came in by elements, as fp32 (putting elements of 16
// bits together again costs more than the registers)
template <Lay L, class T> struct Held {
    float e[8];
    __device__ __forceinline__ void load(const T *row, int i, int width) {
        const bool all = whole<L>(i, width);
#pragma unroll
        for (int k = 0; k < 8; k += L == kPairs ? 2 : 1) {
            const T *at = row + i + place<L>(k);
            const bool in = all || inside<L>(i, k, width);
            if (L == kPairs) {
                PairOf<T> p{(T)0.f, (T)0.f};
                if (in) p = *reinterpret_cast<const PairOf<T> *>(at);
                e[k] = (float)p.a;
                e[k + 1] = (float)p.b;
            } else {
                e[k] = in ? (float)*at : 0.f;
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = e[k];
    }
};
template <class T> struct Held<kPieces, T> {
    Raw8<T> raw;
    __device__ __forceinline__ void load(const T *row, int i, int width) {
        const bool in = i < width;
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k)
            raw.w[k] = in ? *reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned char *>(row + i) + 16 * k) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { widen(raw, v); }
};
template <Lay L, class T>
__device__ __forceinline__ void store_chunk(T *row, int i, int width, const float (&v)[8]) {
    if (L == kPieces) {
        if (i >= width) return;
        alignas(16) T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = (T)v[k];
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) *reinterpret_cast<uint4 *>(reinterpret_cast<unsigned char *>(row + i) + 16 * k) = reinterpret_cast<const uint4 *>(e)[k];
        return;
    }
    const bool all = whole<L>(i, width);
#pragma unroll
    for (int k = 0; k < 8; k += L == kPairs ? 2 : 1)
        if (all || inside<L>(i, k, width)) {
            T *at = row + i + place<L>(k);
            if (L == kPairs) *reinterpret_cast<PairOf<T> *>(at) = PairOf<T>{(T)v[k], (T)v[k + 1]};
            else *at = (T)v[k];
        }
}

// Chunk c, eight neighbours from 8 c on, of a row that begins anywhere: the 16-byte pieces of memory that hold it, shifted.
// near: the memory around the row is its neighbours', so that pieces may be read whole at its ends.
__device__ __forceinline__ void shift_words(uint32_t *w, int n, int by, bool yes) {
    if (!yes) return;
#pragma unroll
    for (int k = 0; k < 12; ++k)
        if (k + by < n) w[k] = w[k + by];
}
template <class T>
__device__ __forceinline__ Raw8<T> load_anywhere(const T *row, int c, int width, bool near) {
    constexpr int kPer = 16 / (int)sizeof(T), kWords = sizeof(T) == 4 ? 12 : 8;            // elements of a piece; words of the pieces
    const int i = c * 8, off = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (kPer - 1)), begin = i - off;
    Raw8<T> r;
    uint32_t *out = &r.w[0].x;
    if (i >= width) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) r.w[k] = make_uint4(0, 0, 0, 0);
        return r;
    }
    if (near || (begin >= 0 && begin + kWords * 4 / (int)sizeof(T) <= width)) {
        uint4 piece[kWords / 4];
#pragma unroll
        for (int k = 0; k < kWords / 4; ++k)
            piece[k] = k < kWords / 4 - 1 || off ? reinterpret_cast<const uint4 *>(row + begin)[k] : make_uint4(0, 0, 0, 0);
        uint32_t w[kWords + 1];
#pragma unroll
        for (int k = 0; k < kWords / 4; ++k) { w[4 * k] = piece[k].x; w[4 * k + 1] = piece[k].y; w[4 * k + 2] = piece[k].z; w[4 * k + 3] = piece[k].w; }
        w[kWords] = 0;
        const int words = off * (int)sizeof(T) / 4;
        shift_words(w, kWords, 2, words & 2);
        shift_words(w, kWords, 1, words & 1);
        if (sizeof(T) == 2) {
            const int bits = 16 * (off & 1);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = __funnelshift_r(w[k], w[k + 1], bits);
        } else {
            uint32_t *more = &r.w[sizeof(T) / 2 - 1].x;
#pragma unroll
            for (int k = 0; k < 4; ++k) { out[k] = w[k]; more[k] = w[4 + k]; }
        }
        if (i + 8 > width) {
#pragma unroll
            for (int k = 1; k < 8; ++k)
                if (i + k >= width) {
                    if (sizeof(T) == 4) (k < 4 ? out[k & 3] : (&r.w[sizeof(T) / 2 - 1].x)[k & 3]) = 0;
                    else out[k >> 1] &= k & 1 ? 0xffffu : 0u;
                }
        }
    } else {
        alignas(16) T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = i + k < width ? row[i + k] : (T)0.f;
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) r.w[k] = reinterpret_cast<const uint4 *>(e)[k];
    }
    return r;
}

// A chunk of a vector of any of the three types by elements (weights: the same for every row, so that they come from the caches)
template <Lay L, class T>
__device__ __forceinline__ void load_elements(const void *vector, int i, int width, float (&v)[8]) {
    const T *from = reinterpret_cast<const T *>(vector);
    const bool all = whole<L>(i, width);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = all || inside<L>(i, k, width) ? (float)from[i + place<L>(k)] : 0.f;
}
template <Lay L>
__device__ __forceinline__ void load_any(const void *vector, int dtype, int i, int width, float (&v)[8]) {
    if (dtype == JQ_BF16) load_elements<L, __nv_bfloat16>(vector, i, width, v);
    else if (dtype == JQ_F16) load_elements<L, __half>(vector, i, width, v);
    else load_elements<L, float>(vector, i, width, v);
}

// Two fp32 operations in one instruction, each rounded as by itself
struct Two { float x, y; };
__device__ __forceinline__ Two add2(Two a, Two b) {
    asm("{ .reg .b64 a, b; mov.b64 a, {%0, %1}; mov.b64 b, {%2, %3}; add.rn.f32x2 a, a, b; mov.b64 {%0, %1}, a; }" : "+f"(a.x), "+f"(a.y) : "f"(b.x), "f"(b.y));
    return a;
}
__device__ __forceinline__ Two fma2(Two a, float f, Two c) {             // a * f + c
    asm("{ .reg .b64 a, c, f; mov.b64 a, {%0, %1}; mov.b64 f, {%4, %4}; mov.b64 c, {%2, %3}; fma.rn.f32x2 a, a, f, c; mov.b64 {%0, %1}, a; }"
        : "+f"(a.x), "+f"(a.y) : "f"(c.x), "f"(c.y), "f"(f));
    return a;
}

// Rotation of 128 neighbours: 16 / A lanes with 8 A of them each, in the order of stages (strides 1, 2, .., 64; sums in the lower place,
// differences in the upper) of fwht128_warp, so that both give the same bits.  Differences, and sums between lanes, are fused multiply-adds
// with 1 or -1, which round as the sum or the difference does, so that all stages but the first take two values at once.
// The shuffles bound it: four per value at A = 1, two at A = 4.
template <int A>
__device__ __forceinline__ void rotate128(float (&v)[A][8], int lane) {
    Two t[4 * A];
#pragma unroll
    for (int i = 0; i < 4 * A; ++i) {
        const float a = v[i >> 2][2 * i & 7], b = v[i >> 2][(2 * i + 1) & 7];
        t[i] = Two{a + b, a - b};
    }
#pragma unroll
    for (int m = 1; m < 4 * A; m <<= 1)
#pragma unroll
        for (int i = 0; i < 4 * A; ++i)
            if (!(i & m)) {
                const Two a = t[i], b = t[i | m];
                t[i] = add2(a, b);
                t[i | m] = fma2(b, -1.f, a);
            }
#pragma unroll
    for (int m = 1; m < 16 / A; m <<= 1) {
        const float sign = (lane & m) ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 4 * A; ++i) {
            const Two o{__shfl_xor_sync(0xffffffffu, t[i].x, m), __shfl_xor_sync(0xffffffffu, t[i].y, m)};
            t[i] = fma2(t[i], sign, o);
        }
    }
#pragma unroll
    for (int i = 0; i < 4 * A; ++i) {
        v[i >> 2][2 * i & 7] = t[i].x * 0.08838834764831845f;
        v[i >> 2][(2 * i + 1) & 7] = t[i].y * 0.08838834764831845f;
    }
}

// Bits of the largest |v|; NaN is above infinity.
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}
// The same of rotated values, by a maximum that keeps a NaN: one may come up beside finite values where the rotation's sums leave fp32's range
// (infinities of one sign that meet), with no infinity left in the block.
template <int A>
__device__ __forceinline__ uint32_t largest_rotated(const float (&v)[A][8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < A; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[j][k])));
    return __float_as_uint(m) & 0x7fffffffu;
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
    // Codes of eight neighbours from i on
    __device__ __forceinline__ void store(int8_t *row, int i, int width, const float (&v)[8]) const {
        const uint2 q = eight(v);
        if (i + 8 <= width) *reinterpret_cast<uint2 *>(row + i) = q;
        else
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k < width) row[i + k] = (int8_t)((k < 4 ? q.x : q.y) >> 8 * (k & 3));
    }
    // of a chunk that lies as L says
    template <Lay L>
    __device__ __forceinline__ void store_as(int8_t *row, int i, int width, const float (&v)[8]) const {
        const uint2 q = eight(v);
        if (L == kPieces) {
            if (i < width) *reinterpret_cast<uint2 *>(row + i) = q;
            return;
        }
        const bool all = whole<L>(i, width);
#pragma unroll
        for (int k = 0; k < 8; k += L == kPairs ? 2 : 1)
            if (all || inside<L>(i, k, width)) {
                const uint32_t b = (k < 4 ? q.x : q.y) >> 8 * (k & 3);
                if (L == kPairs) *reinterpret_cast<uint16_t *>(row + i + place<L>(k)) = (uint16_t)b;
                else row[i + place<L>(k)] = (int8_t)b;
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

inline int chunks_of(int width, Lay l) { return l == kPieces ? (width + 7) / 8 : (width + 255) / 256 * 32; }

// A row's chunks over threads.  Up to 128 chunks a warp has them all and needs no barrier; longer rows have a block, with `many` chunks
// per thread (loads in flight together, few warps at the barriers) unless rows are so few that latency counts: then one.
inline Cut cut_of(int chunks, int rows, int sms, int many) {
    if (chunks <= 128 && (rows > 2 * sms || chunks <= 32)) return Cut{(chunks + 31) / 32, 0};
    const int per = chunks > 2048 ? 4 : rows > 2 * sms || chunks > 1024 ? many : 1;
    const int threads = ((chunks + per - 1) / per + 31) / 32 * 32;
    return Cut{per, threads < 1024 ? threads : 1024};
}

inline bool aligned(const void *p, long long stride, int size) {
    return jq_aligned16(p) && stride * size % 16 == 0;
}

}  // namespace jq8
