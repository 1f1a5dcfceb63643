// The 8-bit key/value cache: how codes lie in a block, what they stand for, and what its kernels share (sm_100a).
//
// A block holds T tokens (16, 32, 64 or 128) of one key head: T * D codes of a byte each for the keys and as many for the
// values, and one fp32 scale for each.  Codes lie in the order in which a warp's matrix instructions (m16n8k16) take
// them as their 16-row operand, K of S^T = K Q^T and V^T of O^T = V^T P^T, so that a lane's 16 bytes are what it multiplies and
// no code is shuffled or transposed:
//   groups of 16 tokens, in a group chunks of 32 values (512 bytes), in a chunk 32 places of 16 bytes;
//   keys:   place (g, t) holds values 8t..8t+7 of the tokens k and k + 2, k = 4 (g / 2) + g % 2;
//   values: place (g, t) holds tokens 4t..4t+3 of the values g, g + 8, g + 16, g + 24
// (g = place / 4, t = place % 4).  A lane gets the scores of the keys that its place names (kv_attend.cu); prompts turn the same 16 bytes
// into operands in shared memory (kv_prompt.cu).
#pragma once
#include "tc.cuh"

namespace jqkv {

constexpr float kTopInt8 = 127.f, kTopE4m3 = 448.f;
constexpr float kLeastMax = 8.673617379884035e-19f;   // 2^-60: the least maximum that a scale is made of, so that its reciprocal is finite
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__host__ __device__ __forceinline__ int key_offset(int token, int d, int D) {
    const int kk = token & 15, place = (2 * (kk >> 2) + (kk & 1)) * 4 + ((d & 31) >> 3);
    return (token >> 4) * 16 * D + (d >> 5) * 512 + place * 16 + ((kk >> 1) & 1) * 8 + (d & 7);
}
__host__ __device__ __forceinline__ int value_offset(int token, int d, int D) {
    const int kk = token & 15, place = (d & 7) * 4 + (kk >> 2);
    return (token >> 4) * 16 * D + (d >> 5) * 512 + place * 16 + ((d & 31) >> 3) * 4 + (kk & 3);
}

// Four codes -> four fp16 values at scale 1, exact.  int8 codes are q + 128: a byte b under the exponent of 1024 is the
// fp16 number 1024 + b.
template <bool E4M3>
__device__ __forceinline__ void codes_to_h4(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (E4M3) {
        asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), bias);
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    }
}

// The sequences of a call.  Everything here is on the device and not looked at by the host: tokens in [0, length) of sequence i
// lie in the blocks table[i][0], table[i][1], ...; its new tokens (queries, or keys to be written) are the rows
// starts[i] .. starts[i + 1] - 1 of the call's tensors and sit at the positions length - n .. length - 1.
struct Batch {
    const int32_t *table, *lengths, *starts;
    int S, width, table_stride, tokens, each;      // each: new tokens of every sequence where starts is null
    int T, shift, blocks;                          // tokens of a block: T = 2^shift

    __device__ __forceinline__ int length(int i) const {
        const int n = lengths[i];
        return n < 0 ? 0 : (n > width * T ? width * T : n);
    }
    // New tokens; 0 where starts does not describe rows of the call's tensors.
    __device__ __forceinline__ int count(int i, int &row0) const {
        if (!starts) {
            row0 = i * each;
            return each;
        }
        const int a = starts[i], b = starts[i + 1];
        row0 = a;
        return a < 0 || b > tokens || b <= a ? 0 : b - a;
    }
    // Block of a sequence's position, -1 where the table does not name one of the pool.
    __device__ __forceinline__ int block(int i, int position) const {
        const int id = table[(size_t)i * table_stride + (position >> shift)];
        return (unsigned)id < (unsigned)blocks ? id : -1;
    }
};

}  // namespace jqkv
