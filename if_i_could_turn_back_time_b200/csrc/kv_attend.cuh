// What the two attention kernels over the 8-bit cache share: arguments, rounding, outputs and the sum of parts.
#pragma once
#include "kv.cuh"

namespace jqkv {

struct AttendArgs {
    Batch b;
    const void *q;
    void *out;
    float *lse;
    long long st, sh;              // elements of q between tokens and heads
    const uint8_t *keys, *values;
    const float *ks, *vs;
    int H, G, window, dtype, least;   // least: units that a CTA takes at least
    float scale;                   // of the scores, times log2(e)
    int *status;
    int *counters;                 // one per CTA: parts of the pair that begins in it and is done elsewhere too
    float *parts;                  // two per CTA: sums, [rows] maxima, [rows] weights (each kernel has an order of its own)
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float lse_of(float m, float l) { return l > 0.f ? (m + log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l); }

// e with amax 2^-e in [2^14, 2^15), as far as 2^e and 2^-e are normal fp32 numbers: every finite row of bf16 is in fp16's range then
// (a row of 2^-126 and less ends below 1).  0 for a row of zeros or with an infinity.
__device__ __forceinline__ int query_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax) & 0x7fffffffu;
    return bits == 0 || bits >= 0x7f800000u ? 0 : max((int)(bits >> 23) - 127 - 14, -126);
}

// First key that a query at this position sees.
__device__ __forceinline__ int first_seen(const AttendArgs &p, int position) {
    return p.window > 0 && position >= p.window ? position - p.window + 1 : 0;
}

// Outputs from element `at` on: v times f, rounded once.
__device__ __forceinline__ uint32_t pack_out(const AttendArgs &p, float a, float b) {
    if (p.dtype == JQ_F16) return pack_h2(a, b);
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&x);
}
__device__ __forceinline__ void store4(const AttendArgs &p, size_t at, const float4 &v, float f) {
    *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.out) + at) = make_uint2(pack_out(p, v.x * f, v.y * f), pack_out(p, v.z * f, v.w * f));
}
__device__ __forceinline__ void store8(const AttendArgs &p, size_t at, const float (&v)[8], float f) {
    *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p.out) + at) =
        make_uint4(pack_out(p, v[0] * f, v[1] * f), pack_out(p, v[2] * f, v[3] * f), pack_out(p, v[4] * f, v[5] * f), pack_out(p, v[6] * f, v[7] * f));
}
// What the sums of a row are divided by; 0 where it saw nothing, NaN stays.
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

// (m, l, v) += another part of the row, both relative to their own m
__device__ __forceinline__ void add_part(float &m, float &l, float4 &v, float mw, float lw, const float4 &y) {
    const float top = fmaxf(m, mw), ref = top == -INFINITY ? 0.f : top;
    const float a = ex2(m - ref), b = ex2(mw - ref);
    v.x = fmaf(v.x, a, y.x * b); v.y = fmaf(v.y, a, y.y * b); v.z = fmaf(v.z, a, y.z * b); v.w = fmaf(v.w, a, y.w * b);
    l = fmaf(l, a, lw * b);
    m = top;
}

// Whole quotients; most operands have 32 bits, whose division is short.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// `total` units dealt to W CTAs: the first `extra` have one more than the others.
struct Shares {
    long long base;
    int extra;
    __device__ __forceinline__ Shares(long long total, int W) : base(quotient(total, W)), extra((int)(total - base * W)) {}
    __device__ __forceinline__ long long first(int w) const { return base * w + min(w, extra); }
    __device__ __forceinline__ int owner(long long unit) const {
        const long long longer = extra * (base + 1);
        return unit < longer ? (int)quotient(unit, base + 1) : extra + (int)quotient(unit - longer, base);
    }
};

// Prompts (kv_prompt.cu): rows of a CTA, CTAs, bytes of their parts, launch.
constexpr int kPromptRows = 256;
static inline int prompt_grid() { return jq_sm_count() < kJqCounters ? jq_sm_count() : kJqCounters; }
size_t prompt_workspace(int D);
int prompt_launch(const AttendArgs &a, int D, bool e4m3, cudaStream_t st);

}  // namespace jqkv
