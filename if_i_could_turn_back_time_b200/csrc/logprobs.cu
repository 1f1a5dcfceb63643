// Log probabilities of given tokens, entropies and the strongest alternatives of rows of logits, in one pass over the row.
#include "common.cuh"

namespace jqlp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kFull = 0xffffffffu;

struct Args {
    const void *x;
    long long stride;                          // elements between rows
    const long long *tokens;
    float *logprob, *entropy, *top_logprob;
    long long *top_token;
    int rows, vocab, k, parts, chunk;          // chunk: elements of a part, a multiple of 2048
    int *counters;                             // one per row
    float *sums;                               // three per part
    unsigned long long *lists;                 // 32 per part
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A value and its index as a whole number: larger values first, the lower index first among equals (0 and -0 are equal; NaN is
// above everything).
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
    uint32_t u = __float_as_uint(x + 0.f);
    if (x != x) u = 0x7fffffffu;
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (unsigned long long)u << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// Lane i of a warp holds the i-th largest key.  Keys `other`, in order too, are merged in: of 64 keys the 32 largest stay.
__device__ __forceinline__ unsigned long long max64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long merge_sorted(unsigned long long list, unsigned long long other, int lane) {
    const unsigned long long turned = __shfl_sync(kFull, other, 31 - lane);
    unsigned long long v = max64(list, turned);            // the 32 largest, rising and then falling at most once
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long w = __shfl_xor_sync(kFull, v, o);
        v = ((lane & o) == 0) == (v > w) ? v : w;
    }
    return v;
}
__device__ __forceinline__ unsigned long long sort_warp(unsigned long long v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const unsigned long long w = __shfl_xor_sync(kFull, v, o);
            const bool falling = (lane & size) == 0 || size == 32;
            v = (((lane & o) == 0) == falling) == (v > w) ? v : w;
        }
    return v;
}
__device__ __forceinline__ unsigned long long insert(unsigned long long list, unsigned long long key, int lane) {
    const int at = __popc(__ballot_sync(kFull, list > key));
    const unsigned long long up = __shfl_up_sync(kFull, list, 1);
    return lane < at ? list : (lane == at ? key : up);
}

// m: the largest value so far; l = sum of e^(x - m); u = sum of e^(x - m) (x - m)
struct Sums {
    float m, l, u;
    __device__ __forceinline__ void to(float top) {        // the same sums relative to a larger (or equal) m
        if (top == m) return;
        const float d = m - top, f = l > 0.f ? ex2(d * kLog2e) : (l == 0.f ? 0.f : l);
        u = l > 0.f && f > 0.f ? f * fmaf(l, d, u) : (l != l ? l : 0.f);
        l *= f;
        m = top;
    }
    __device__ __forceinline__ void add(Sums o) {
        const float top = fmaxf(m, o.m);
        to(top);
        o.to(top);
        l += o.l;
        u += o.u;
    }
};

template <class T> __device__ __forceinline__ float as_float(T x) { return (float)x; }

template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ Args p) {
    constexpr int V = 16 / sizeof(T);                      // elements of a load
    constexpr int L = 4;                                   // loads of a step
    __shared__ Sums s_sums[kWarps];
    __shared__ unsigned long long s_lists[TOP ? kWarps : 1][32];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const T *x = reinterpret_cast<const T *>(p.x) + (long long)row * p.stride;
    const int begin = min(p.vocab, part * p.chunk), end = min(p.vocab, begin + p.chunk);

    Sums s{-INFINITY, 0.f, 0.f};
    unsigned long long list = 0;                           // (below every key)
    float least = -INFINITY;                               // the k-th value of this warp's list, and its index
    uint32_t least_at = 0xffffffffu;

    auto take = [&](const float (&v)[V], uint32_t at, int count) {       // `count` values from index `at` on; warp-uniform flow where TOP
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, v[e]);
        if (top > s.m) s.to(top);
        const float m = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = v[e] - m, w = ex2(d * kLog2e);
            s.l += w;
            s.u = fmaf(w, fmaxf(d, -1e30f), s.u);          // (0 times -infinity is 0)
        }
        if (TOP) {
            const bool better = count > 0 && (top > least || (top == least && at < least_at));
            if (__any_sync(kFull, better)) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const unsigned long long bar = __shfl_sync(kFull, list, p.k - 1);
                    unsigned long long key = e < count ? key_of(v[e], at + e) : 0;
                    if (key <= bar) key = 0;
                    unsigned hits = __ballot_sync(kFull, key != 0);
                    if (__popc(hits) > 6) {
                        list = merge_sorted(list, sort_warp(key, lane), lane);
                    } else {
                        while (hits) {
                            list = insert(list, __shfl_sync(kFull, key, __ffs(hits) - 1), lane);
                            hits &= hits - 1;
                        }
                    }
                }
                const unsigned long long bar = __shfl_sync(kFull, list, p.k - 1);
                if (bar) {
                    least = value_of(bar);
                    least_at = ~(uint32_t)bar;
                }
            }
        }
    };

    // values before the first 16-byte boundary and behind the last are taken one by one (a thread has at most one of them)
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x + begin) & 15u)) % 16 / sizeof(T)), end - begin);
    const int body = (end - begin - head) / V, tail0 = begin + head + body * V;
    if (warp == 0) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = -INFINITY;
        const int at = lane < head ? begin + lane : tail0 + lane - head;
        const bool there = lane < head + (end - tail0);
        if (there) v[0] = as_float(x[at]);
        take(v, at, there ? 1 : 0);
    }
    const uint4 *xb = reinterpret_cast<const uint4 *>(x + begin + head);
    for (int i0 = warp * 32; i0 < body; i0 += kThreads * L) {
        uint4 raw[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int i = i0 + j * kThreads + lane;
            if (i < body) raw[j] = __ldcs(xb + i);
        }
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int i = i0 + j * kThreads + lane;
            if (i0 + j * kThreads >= body) break;
            float v[V];
            const T *e = reinterpret_cast<const T *>(&raw[j]);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = i < body ? as_float(e[k]) : -INFINITY;
            take(v, (uint32_t)(begin + head + i * V), i < body ? V : 0);
        }
    }

    // ---- the block's sums and list
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        s.add(Sums{__shfl_xor_sync(kFull, s.m, o), __shfl_xor_sync(kFull, s.l, o), __shfl_xor_sync(kFull, s.u, o)});
    if (lane == 0) s_sums[warp] = s;
    if (TOP) s_lists[warp][lane] = list;
    __syncthreads();
    if (warp != 0) return;                                 // (what is left is one warp's work)
    s = s_sums[0];
    for (int w = 1; w < kWarps; ++w) s.add(s_sums[w]);
    if (TOP)
        for (int w = 1; w < kWarps; ++w) list = merge_sorted(list, s_lists[w][lane], lane);
    if (p.parts > 1) {
        const size_t mine = (size_t)row * p.parts + part;
        if (lane == 0) {
            p.sums[mine * 3] = s.m;
            p.sums[mine * 3 + 1] = s.l;
            p.sums[mine * 3 + 2] = s.u;
        }
        if (TOP) p.lists[mine * 32 + lane] = list;
        __threadfence();
        __syncwarp();
        if (lane == 0) {
            s_last = atomicAdd(p.counters + row, 1) == p.parts - 1;
            if (s_last) p.counters[row] = 0;
        }
        __syncwarp();
        if (!s_last) return;
        __threadfence();
        // the row's last part adds all of them, in their order
        const size_t first = (size_t)row * p.parts;
        s = Sums{-INFINITY, 0.f, 0.f};
        list = 0;
        for (int w = 0; w < p.parts; ++w) {
            const float *o = p.sums + (first + w) * 3;
            s.add(Sums{__ldcg(o), __ldcg(o + 1), __ldcg(o + 2)});
            if (TOP) list = merge_sorted(list, __ldcg(p.lists + (first + w) * 32 + lane), lane);
        }
    }
    const float log_l = logf(s.l);
    auto logprob = [&](float v) { return s.m == -INFINITY ? (s.l == 0.f ? -INFINITY : s.l) : v - s.m - log_l; };
    if (lane == 0) {
        const long long token = p.tokens[row];
        p.logprob[row] = token < 0 ? 0.f : (token >= p.vocab ? __int_as_float(0x7fffffff) : logprob(as_float(x[token])));
        if (p.entropy) p.entropy[row] = s.m == -INFINITY && s.l == 0.f ? 0.f : log_l - s.u / s.l;
    }
    if (TOP && lane < p.k) {
        p.top_logprob[(size_t)row * p.k + lane] = logprob(value_of(list));
        p.top_token[(size_t)row * p.k + lane] = (long long)(uint32_t)~(uint32_t)list;
    }
}

// Parts of a row: one where the rows fill the chip by themselves.
static int parts_of(int rows, int vocab) {
    const int fill = 4 * jq_sm_count() < kJqCounters ? 4 * jq_sm_count() : kJqCounters;
    const int steps = (vocab + 2047) / 2048;
    int parts = rows >= fill ? 1 : fill / rows;
    return parts < steps ? parts : steps;
}

}  // namespace jqlp

using namespace jqlp;

extern "C" size_t jq_token_logprobs_workspace_bytes(int rows, int vocab) {
    if (rows <= 0 || vocab <= 0) return 0;
    const size_t parts = (size_t)parts_of(rows, vocab);
    if (parts == 1) return 0;
    return kJqData + (size_t)rows * parts * (32 * 8 + 12);
}

extern "C" int jq_token_logprobs(const void *logits, int64_t row_stride, int rows, int vocab, int dtype, const int64_t *tokens,
                                 float *logprob, float *entropy_or_null, int top, float *top_logprob_or_null,
                                 int64_t *top_token_or_null, void *workspace, size_t workspace_bytes, jq_stream_t stream) {
    if (rows < 0 || vocab <= 0 || top < 0 || top > 32 || top > vocab) return JQ_ERR_BAD_SHAPE;
    if (dtype < 0 || dtype > 2) return JQ_ERR_BAD_DTYPE;
    if (rows == 0) return JQ_OK;
    if (!logits || !tokens || !logprob || (top && (!top_logprob_or_null || !top_token_or_null))) return JQ_ERR_NULL_PTR;
    if (vocab > (1 << 30) || row_stride < 0) return JQ_ERR_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(logits) & (dtype == JQ_F32 ? 3u : 1u)) || (reinterpret_cast<uintptr_t>(tokens) & 7u) ||
        (reinterpret_cast<uintptr_t>(top_token_or_null) & 7u) || ((reinterpret_cast<uintptr_t>(logprob) | reinterpret_cast<uintptr_t>(entropy_or_null) |
        reinterpret_cast<uintptr_t>(top_logprob_or_null)) & 3u) || (reinterpret_cast<uintptr_t>(workspace) & 127u))
        return JQ_ERR_BAD_ALIGN;
    const size_t need = jq_token_logprobs_workspace_bytes(rows, vocab);
    if (need && !workspace) return JQ_ERR_NULL_PTR;
    if (need > workspace_bytes) return JQ_ERR_WORKSPACE;
    Args a{};
    a.x = logits; a.stride = row_stride; a.tokens = reinterpret_cast<const long long *>(tokens);
    a.logprob = logprob; a.entropy = entropy_or_null; a.top_logprob = top_logprob_or_null;
    a.top_token = reinterpret_cast<long long *>(top_token_or_null);
    a.rows = rows; a.vocab = vocab; a.k = top; a.parts = parts_of(rows, vocab);
    a.chunk = ((vocab + a.parts - 1) / a.parts + 2047) / 2048 * 2048;
    unsigned char *ws = reinterpret_cast<unsigned char *>(workspace);
    if (a.parts > 1) {
        a.counters = reinterpret_cast<int *>(ws + kJqHeader);
        a.lists = reinterpret_cast<unsigned long long *>(ws + kJqData);
        a.sums = reinterpret_cast<float *>(a.lists + (size_t)rows * a.parts * 32);
    }
    const long long grid = (long long)rows * a.parts;
    if (grid > 0x7fffffffLL) return JQ_ERR_BAD_SHAPE;
    void (*const kernels[3][2])(const Args) = {{logprobs_kernel<float, false>, logprobs_kernel<float, true>},
                                               {logprobs_kernel<__half, false>, logprobs_kernel<__half, true>},
                                               {logprobs_kernel<__nv_bfloat16, false>, logprobs_kernel<__nv_bfloat16, true>}};
    kernels[dtype][top > 0]<<<(unsigned)grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    return jq_launch_status();
}
