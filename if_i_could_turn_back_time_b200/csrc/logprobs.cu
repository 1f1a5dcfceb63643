// Log probabilities of given tokens, entropies and the strongest alternatives of rows of logits, in one pass over the row.
//
// Bound by reading the logits where there are many: 1024 rows of 131072 fp32, 537 MB: 94 us, 5.7 TB/s; 2047 rows of 32003 bf16, 131 MB: 33 us, 4 TB/s (2.3
// waves of CTAs).  64 rows of 131072 with 20 alternatives take 16 us, 3 of them reading: the rest are barriers and the join of nine parts a row.
#include "common.cuh"

namespace jqlp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kFull = 0xffffffffu;
constexpr int kCandidates = 1024;              // keys that are ranked at most

struct Args {
    const void *x;
    long long stride;                          // elements between rows
    const long long *tokens;
    float *logprob, *entropy, *top_logprob;
    long long *top_token;
    int rows, vocab, k, parts, chunk;          // chunk: elements of a part, a multiple of 512
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
// above everything, but only a NaN that has a large number beside it in its 16 bytes is looked at: the alternatives of a row with a
// NaN are some of its tokens).
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

// Two fp32 values in a register pair
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair2(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 16 bytes of logits
template <class T> struct Vec;
template <> struct Vec<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
    }
};
template <> struct Vec<__half> {
    static constexpr int V = 8;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

__device__ __forceinline__ uint32_t ordered(float x) {      // larger values, larger numbers; NaN is not asked for
    const uint32_t u = __float_as_uint(x + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A part of a row: its elements, and how threads take them: those before the first 16-byte boundary and behind the last one by one,
// by the first warp's lanes; the others 16 bytes at a time, thread by thread.
template <class T>
struct Part {
    static constexpr int V = Vec<T>::V;
    const T *x;
    int begin, head, body, tail0, end;
    __device__ __forceinline__ Part(const T *row, int b, int e) : x(row), begin(b), end(e) {
        head = min((int)((16 - (reinterpret_cast<uintptr_t>(row + b) & 15u)) % 16 / sizeof(T)), e - b);
        body = (e - b - head) / V;
        tail0 = b + head + body * V;
    }
    __device__ __forceinline__ int single(int tid) const {   // index of the thread's single element, -1: none
        return tid < head ? begin + tid : (tid < head + end - tail0 ? tail0 + tid - head : -1);
    }
    __device__ __forceinline__ const uint4 *vectors() const { return reinterpret_cast<const uint4 *>(x + begin + head); }
    __device__ __forceinline__ int index(int vector) const { return begin + head + vector * V; }
};

// The k largest keys of the part, the plain way: every warp keeps a sorted list.  Any number of equal values; used where the candidates of
// the quick way (below) are too many.
template <class T>
__device__ __noinline__ void scan_lists(const Part<T> part, int k, unsigned long long (*lists)[32], unsigned long long *out) {
    constexpr int V = Part<T>::V;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long list = 0, bar = 0;
    auto take = [&](unsigned long long key) {
        if (key <= bar) key = 0;
        unsigned hits = __ballot_sync(kFull, key != 0);
        if (!hits) return;
        if (__popc(hits) > 6) {
            list = merge_sorted(list, sort_warp(key, lane), lane);
        } else {
            while (hits) {
                list = insert(list, __shfl_sync(kFull, key, __ffs(hits) - 1), lane);
                hits &= hits - 1;
            }
        }
        bar = __shfl_sync(kFull, list, k - 1);
    };
    if (warp == 0) {
        const int at = part.single(lane);
        take(at >= 0 ? key_of((float)part.x[at], at) : 0);
    }
    for (int i0 = warp * 32; i0 < part.body; i0 += kThreads) {
        const int i = i0 + lane;
        float v[V];
        if (i < part.body) Vec<T>::values(part.vectors()[i], v);
#pragma unroll
        for (int e = 0; e < V; ++e) take(i < part.body ? key_of(v[e], part.index(i) + e) : 0);
    }
    lists[warp][lane] = list;
    __syncthreads();
    if (warp == 0) {
        for (int w = 1; w < kWarps; ++w) list = merge_sorted(list, lists[w][lane], lane);
        out[lane] = list;
    }
    __syncthreads();
}

// The 32 largest of `count` different keys in falling order, 0 behind them: a key's place is the number of keys above it.
__device__ __forceinline__ void rank_keys(const unsigned long long *keys, int count, unsigned long long *out) {
    if (threadIdx.x < 32) out[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const unsigned long long mine = keys[i];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) above += keys[j] > mine;
        if (above < 32) out[above] = mine;
    }
    __syncthreads();
}

// Top tokens the quick way.  A thread knows the largest of its elements.  With j = ceil(k / 8), the j-th largest of a warp's 32 such
// values, and the least of these over the 8 warps, is a bound that at least 8 j >= k elements of the part reach; it is raised by halving
// while k threads' largest values reach it.  Only those threads look again, nearly always at the one 16-byte piece that had their largest, and
// what reaches the bound (little more than k of random values) is ranked.
template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ Args p) {
    constexpr int V = Vec<T>::V;
    constexpr int L = 32 / V;                              // loads of a step: 32 elements a thread
    __shared__ float s_l[kWarps], s_u[kWarps];
    __shared__ uint32_t s_top[kWarps], s_bar[kWarps];
    __shared__ unsigned long long s_keys[TOP ? kCandidates : 1], s_list[32];
    __shared__ int s_count, s_threads, s_last;
    __shared__ unsigned char s_hot[TOP ? kThreads : 1];
    static_assert(!TOP || kCandidates >= kWarps * 32, "the lists of scan_lists lie there too");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.parts, at_part = blockIdx.x % p.parts;
    const T *x = reinterpret_cast<const T *>(p.x) + (long long)row * p.stride;
    const int begin = min(p.vocab, at_part * p.chunk);
    const Part<T> part(x, begin, min(p.vocab, begin + p.chunk));

    // ---- one pass: m, the largest value so far; l and u, sums of e^(x - m) and e^(x - m) (x - m)
    Sums s{-INFINITY, 0.f, 0.f};
    float second = -INFINITY;                              // the largest value outside the piece that has the largest, and that piece
    int piece = -1;
    auto take = [&](const float (&v)[V], int i) {
        float top = v[0];
#pragma unroll
        for (int e = 1; e < V; ++e) top = fmaxf(top, v[e]);
        if (top > s.m) {
            if (TOP) {
                second = s.m;
                piece = i;
            }
            s.to(top);
        } else if (TOP) {
            second = fmaxf(second, top);
        }
        const float m = s.m == -INFINITY ? 0.f : -s.m;
        const uint64_t m2 = pair2(m, m), scale = pair2(kLog2e, kLog2e);
        uint64_t l = pair2(s.l, 0.f), u = pair2(s.u, 0.f);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const uint64_t d = add2(pair2(v[e], v[e + 1]), m2);
            const float2 y = unpair2(mul2(d, scale)), f = unpair2(d);
            const uint64_t w = pair2(ex2(y.x), ex2(y.y));
            l = add2(l, w);
            u = fma2(w, pair2(fmaxf(f.x, -1e30f), fmaxf(f.y, -1e30f)), u);       // (0 times -infinity is 0)
        }
        const float2 a = unpair2(l), b = unpair2(u);
        s.l = a.x + a.y;
        s.u = b.x + b.y;
    };
    const uint4 *const xb = part.vectors();
    for (int i0 = tid; i0 < part.body; i0 += kThreads * L) {
        uint4 raw[L];
#pragma unroll
        for (int j = 0; j < L; ++j)
            if (i0 + j * kThreads < part.body) raw[j] = __ldg(xb + i0 + j * kThreads);
#pragma unroll
        for (int j = 0; j < L; ++j)
            if (i0 + j * kThreads < part.body) {
                float v[V];
                Vec<T>::values(raw[j], v);
                take(v, i0 + j * kThreads);
            }
    }
    const int single = part.single(tid);
    if (single >= 0) {
        float v[V];
#pragma unroll
        for (int e = 1; e < V; ++e) v[e] = -INFINITY;
        v[0] = (float)x[single];
        take(v, -1);                                       // (a single value is always looked at again by itself)
    }

    // ---- the block's largest value, and the bound
    uint32_t mine = ordered(s.m);
    const uint32_t warp_top = __reduce_max_sync(kFull, mine);
    if (lane == 0) s_top[warp] = warp_top;
    if (TOP) {
        uint32_t left = mine, bar = warp_top;
        for (int j = (p.k + kWarps - 1) / kWarps; j > 1; --j) {                   // (one lane of those that have the largest leaves)
            const unsigned has = __ballot_sync(kFull, left == bar);
            if (lane == __ffs(has) - 1) left = 0;
            bar = __reduce_max_sync(kFull, left);
        }
        if (lane == 0) s_bar[warp] = bar;
        if (tid == 0) s_count = s_threads = 0;
    }
    __syncthreads();
    uint32_t top = s_top[0], bar = s_bar[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
        top = max(top, s_top[w]);
        if (TOP) bar = min(bar, s_bar[w]);
    }
    s.to(value_of((unsigned long long)top << 32));
    float l = jq::warp_sum(s.l), u = jq::warp_sum(s.u);
    if (lane == 0) {
        s_l[warp] = l;
        s_u[warp] = u;
    }
    if (TOP) {
        auto offer = [&](float v, int at) {
            const unsigned long long key = key_of(v, at);
            if ((uint32_t)(key >> 32) < bar) return;
            const int i = atomicAdd(&s_count, 1);
            if (i < kCandidates) s_keys[i] = key;
        };
        // a better bound by halving: as many threads as may be reach it, as long as these are at least k
        uint32_t high = top;
        int threads = __syncthreads_count(mine >= bar);
        for (int i = 0; i < 16 && bar < high && threads > p.k + 8; ++i) {
            const uint32_t mid = bar + (high - bar + 1) / 2;
            const int c = __syncthreads_count(mine >= mid);
            if (c >= p.k) {
                bar = mid;
                threads = c;
            } else {
                high = mid - 1;
            }
        }
        // what reaches it: a thread whose other pieces do not looks at one piece again; the others' pieces go to all threads
        auto look = [&](int i) {
            float v[V];
            Vec<T>::values(__ldg(xb + i), v);
            float most = v[0];
#pragma unroll
            for (int e = 1; e < V; ++e) most = fmaxf(most, v[e]);
            if (ordered(most) < bar) return;
#pragma unroll
            for (int e = 0; e < V; ++e) offer(v[e], part.index(i) + e);
        };
        if (mine >= bar) {
            if (ordered(second) >= bar) s_hot[atomicAdd(&s_threads, 1)] = (unsigned char)tid;
            else if (piece >= 0) look(piece);
            if (single >= 0) offer((float)x[single], single);
        }
        __syncthreads();
        const int hot = s_threads, rounds = (part.body + kThreads - 1) / kThreads;
        for (int q = tid; q < hot * rounds; q += kThreads) {
            const int i = s_hot[q % hot] + q / hot * kThreads;
            if (i < part.body) look(i);
        }
    }
    __syncthreads();
    float m = s.m;
    l = u = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        l += s_l[w];
        u += s_u[w];
    }
    if (TOP) {
        const int count = s_count;
        if (count <= kCandidates) rank_keys(s_keys, count, s_list);
        else scan_lists(part, p.k, reinterpret_cast<unsigned long long(*)[32]>(s_keys), s_list);
    }
    if (p.parts > 1) {
        // the row's last part adds all of them, in an order that does not depend on which it is
        const size_t first = (size_t)row * p.parts, own = first + at_part;
        if (tid == 0) {
            p.sums[own * 3] = m;
            p.sums[own * 3 + 1] = l;
            p.sums[own * 3 + 2] = u;
        }
        if (TOP && tid < 32) p.lists[own * 32 + tid] = s_list[tid];
        if (tid < 32) __threadfence();
        __syncthreads();
        if (tid == 0) {
            s_last = atomicAdd(p.counters + row, 1) == p.parts - 1;
            if (s_last) p.counters[row] = 0;
            s_count = 0;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        float pm = -INFINITY, pl = 0.f, pu = 0.f;
        unsigned long long least = 0;                      // the largest of the parts' k-th keys: k keys reach it
        s = Sums{-INFINITY, 0.f, 0.f};
        for (int i = tid; i < p.parts; i += kThreads) {
            const float *o = p.sums + (first + i) * 3;
            pm = __ldcg(o);
            pl = __ldcg(o + 1);
            pu = __ldcg(o + 2);
            s.add(Sums{pm, pl, pu});
            if (TOP) least = max64(least, __ldcg(p.lists + (first + i) * 32 + p.k - 1));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s.add(Sums{__shfl_xor_sync(kFull, s.m, o), __shfl_xor_sync(kFull, s.l, o), __shfl_xor_sync(kFull, s.u, o)});
            if (TOP) least = max64(least, __shfl_xor_sync(kFull, least, o));
        }
        __shared__ Sums s_sums[kWarps];
        __shared__ unsigned long long s_least[kWarps];
        if (lane == 0) {
            s_sums[warp] = s;
            s_least[warp] = least;
        }
        __syncthreads();
        s = s_sums[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            s.add(s_sums[w]);
            if (TOP) least = max64(least, s_least[w]);
        }
        if (TOP) {
            least = max64(least, s_least[0]);
            for (int i = tid; i < p.parts * 32; i += kThreads) {
                const unsigned long long key = __ldcg(p.lists + first * 32 + i);
                if (!key || key < least) continue;
                const int c = atomicAdd(&s_count, 1);
                if (c < kCandidates) s_keys[c] = key;
            }
            __syncthreads();
            const int count = s_count;
            if (count <= kCandidates) {
                rank_keys(s_keys, count, s_list);
            } else if (warp == 0) {                        // (many parts whose lists lie between one another)
                unsigned long long list = 0;
                for (int i = 0; i < p.parts; ++i) list = merge_sorted(list, __ldcg(p.lists + (first + i) * 32 + lane), lane);
                s_list[lane] = list;
                __syncwarp();
            }
        }
        m = s.m;
        l = s.l;
        u = s.u;
    }
    if (warp != 0) return;
    const float log_l = logf(l);
    auto logprob = [&](float v) { return m == -INFINITY ? (l == 0.f ? -INFINITY : l) : v - m - log_l; };
    if (lane == 0) {
        const long long token = p.tokens[row];
        p.logprob[row] = token < 0 ? 0.f : (token >= p.vocab ? __int_as_float(0x7fffffff) : logprob((float)x[token]));
        if (p.entropy) p.entropy[row] = m == -INFINITY && l == 0.f ? 0.f : log_l - u / l;
    }
    if (TOP && lane < p.k) {
        const unsigned long long key = s_list[lane];
        p.top_logprob[(size_t)row * p.k + lane] = logprob(value_of(key));
        p.top_token[(size_t)row * p.k + lane] = (long long)(uint32_t)~(uint32_t)key;
    }
}

constexpr int kStep = 2048;                    // a row has at most one part for so many elements (chunks are rounded to 512)

// Parts of a row: as many as fill the chip where there are few rows, one where the rows fill it by themselves.  (Halves that would fill a
// partly empty last wave cost more than it: 2047 rows of 32003 bf16 33 us whole, 46 us in halves; 1024 of 131072 fp32 108 and 115.)
static int parts_of(int rows, int vocab) {
    const int fill = 4 * jq_sm_count() < kJqCounters ? 4 * jq_sm_count() : kJqCounters;
    const int most = (vocab + kStep - 1) / kStep, parts = rows >= fill ? 1 : fill / rows;
    return parts < most ? parts : most;
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
    a.chunk = ((vocab + a.parts - 1) / a.parts + 511) / 512 * 512;
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
