// Log probabilities of given tokens, the entropy and the best alternatives of
// rows of logits, in one pass over them.
//
// With m = max x, z = sum e^(x - m) and t = sum e^(x - m) (x - m):
//   log p(i) = (x_i - m) - ln z,   entropy = ln z - t / z
// (both terms of the entropy are positive, nothing cancels). Each thread keeps
// (m, z, t) of its share; a new maximum m' turns them into
// (m', z r, (t + z (m - m')) r) with r = e^(m - m'), and the same rule joins
// threads, waves and workgroups in a fixed order, in F32.
//
// The k best are ordered by (value descending, id ascending): one 64-bit key,
// smaller is better. A wave keeps the best key of each lane; the k-th best of
// these 64 (k <= 32) is a bound that k different logits reach, so only keys up to
// it can be among the answer. They go to a queue in LDS, which a short row of
// comparisons (16 logits a lane at a time) leaves alone almost always: about
// 64 ln(64 / (64 - k)) logits reach the bound of the data so far. At the end
// the waves' queues, cut by the best bound, are ranked by counting.
//
// Bound by the read of the logits. A row is split over workgroups where there
// are few rows; the splits' results go to the workspace for a second kernel.
#include "kernels.h"

namespace nuq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.44269504088896340736f;
constexpr uint64_t PAD = ~0ull;  // after every key
constexpr uint32_t THREADS = 256, WAVES = 4, QUEUE = 256;
constexpr int EACH = 16;         // logits a thread holds at a time

__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) {
    uint32_t u = __float_as_uint(v);
    if (v == 0.0f) u = 0;  // -0 ties with +0
    const uint32_t order = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return v != v ? PAD : (uint64_t)~order << 32 | i;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t order = ~(uint32_t)(key >> 32);
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}

struct Stats {
    float m, z, t;
};
// (0 for a share of nothing: m is LOWEST, and the clamp keeps 0 * inf away)
__device__ __forceinline__ Stats rebased(const Stats &s, float m) {
    const float by = fmaxf(s.m - m, -1000.0f), r = __builtin_amdgcn_exp2f(by * LOG2E);
    return {m, s.z * r, (s.t + s.z * by) * r};
}
__device__ __forceinline__ Stats joined(const Stats &a, const Stats &b) {
    const float m = fmaxf(a.m, b.m);
    const Stats x = rebased(a, m), y = rebased(b, m);
    return {m, x.z + y.z, x.t + y.t};
}

__device__ __forceinline__ uint64_t lane_key(uint64_t key, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)key, lane);
}

// The k-th best of a wave's 64 keys (PAD where fewer are real).
__device__ __forceinline__ uint64_t kth_of_lanes(uint64_t key, uint32_t k) {
    uint32_t rank = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) rank += lane_key(key, j) < key;
    const uint64_t at = __ballot(rank == k - 1);
    return at ? lane_key(key, __builtin_ctzll(at)) : PAD;
}

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Keeps the k best of a wave's queue of `count` keys, in order.
__device__ __noinline__ uint32_t shorten(uint64_t *queue, uint32_t count, uint32_t k, uint32_t lane) {
    constexpr int HELD = QUEUE / 64;
    uint64_t mine[HELD];
    uint32_t rank[HELD] = {};
    wave_sync();
#pragma unroll
    for (int i = 0; i < HELD; ++i) mine[i] = lane + 64 * i < count ? queue[lane + 64 * i] : PAD;
    for (uint32_t j = 0; j < count; ++j) {
        const uint64_t other = queue[j];
#pragma unroll
        for (int i = 0; i < HELD; ++i) rank[i] += other < mine[i];
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (mine[i] != PAD && rank[i] < k) queue[rank[i]] = mine[i];
    wave_sync();
    return min(count, k);
}

struct LogprobArgs {
    const void *logits;
    uint64_t stride;
    const int32_t *targets;
    float *logprobs, *entropy;
    uint32_t *ids;
    float *tops;
    uint32_t rows, count, top, splits, span;  // span: vectors of a split
    uint64_t *keys;  // [rows][splits][top]
    float *stats;    // [rows][splits][3]
};

// The row's answer from its statistics; the tops are `list`'s keys by rank.
template <typename T>
__device__ __forceinline__ void finish(const LogprobArgs &a, uint32_t row, const Stats &s, const uint64_t *list,
                                       uint32_t n, uint32_t tid) {
    const float ln_z = logf(s.z);
    if (tid == 0) {
        const uint32_t id = (uint32_t)a.targets[row];
        float lp = __builtin_nanf("");  // no such token
        if (id < a.count) {
            const float x = (float)((const T *)a.logits)[(uint64_t)row * a.stride + id];
            // a row of -inf alone has no distribution: -inf and no entropy
            lp = s.z == 0.0f ? -__builtin_inff() : (x - s.m) - ln_z;
        }
        a.logprobs[row] = lp;
        a.entropy[row] = s.z == 0.0f ? 0.0f : ln_z - s.t / s.z;
    }
    for (uint32_t i = tid; i < n; i += THREADS) {
        const uint64_t mine = list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += list[j] < mine;
        if (rank < a.top) {
            const uint64_t at = (uint64_t)row * a.top + rank;
            a.ids[at] = (uint32_t)mine;
            a.tops[at] = s.z == 0.0f ? -__builtin_inff() : (value_of(mine) - s.m) - ln_z;
        }
    }
    for (uint32_t i = n + tid; i < a.top; i += THREADS) {  // fewer numbers than asked for
        a.ids[(uint64_t)row * a.top + i] = 0xffffffffu;
        a.tops[(uint64_t)row * a.top + i] = -__builtin_inff();
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) logprobs_kernel(LogprobArgs a) {
    constexpr int V = 16 / sizeof(T), VECTORS = EACH / V;
    __shared__ uint64_t queues[WAVES][QUEUE], list[WAVES * QUEUE];
    __shared__ Stats wave_stats[WAVES];
    __shared__ uint64_t wave_bound[WAVES];
    __shared__ uint32_t wave_count[WAVES], listed;
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const T *x = (const T *)a.logits + (uint64_t)row * a.stride;
    // vectors are 16-byte aligned: the first may begin before the row
    const int before = (int)(((uintptr_t)x & 15) / sizeof(T));
    const uint32_t vectors = (uint32_t)((before + (uint64_t)a.count + V - 1) / V);
    const uint32_t end = min(vectors, (split + 1) * a.span);
    uint64_t *queue = queues[wave];

    Stats s = {LOWEST, 0.0f, 0.0f};
    uint64_t best = PAD, bound = PAD;
    float bound_value = -__builtin_inff();
    uint32_t count = 0;
    for (uint32_t base = split * a.span; base < end; base += THREADS * VECTORS) {
        float v[EACH];
#pragma unroll
        for (int u = 0; u < VECTORS; ++u) {
            const uint32_t at = base + u * THREADS + tid;
            const int64_t first = (int64_t)at * V - before;
            if (at < end && first >= 0 && first + V <= (int64_t)a.count) {
                if constexpr (V == 4) {
                    const float4 f = *(const float4 *)(x + first);
                    v[4 * u] = f.x, v[4 * u + 1] = f.y, v[4 * u + 2] = f.z, v[4 * u + 3] = f.w;
                } else {
                    const half8 f = *(const half8 *)(x + first);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[V * u + e] = (float)f[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int64_t i = first + e;
                    v[V * u + e] = at < end && i >= 0 && i < (int64_t)a.count ? (float)x[i] : -__builtin_inff();
                }
            }
        }
        float most = v[0];
#pragma unroll
        for (int e = 1; e < EACH; ++e) most = fmaxf(most, v[e]);
        if (most > s.m) s = rebased(s, most);
        float z = 0.0f, t = 0.0f;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const float d = v[e] - s.m, p = __builtin_amdgcn_exp2f(d * LOG2E);
            z += p;
            t += p * fmaxf(d, -1000.0f);  // 0, not 0 * inf, for a logit of -inf
        }
        s.z += z, s.t += t;
        if (a.top == 0 || !__any(most >= bound_value)) continue;
        // absent places (before and behind the row) have no key
        const auto key = [&](int e) {
            const int64_t i = (int64_t)(base + e / V * THREADS + tid) * V - before + e % V;
            const bool real = base + e / V * THREADS + tid < end && i >= 0 && i < (int64_t)a.count;
            return real ? key_of(v[e], (uint32_t)i) : PAD;
        };
#pragma unroll
        for (int e = 0; e < EACH; ++e) best = min(best, key(e));
        bound = min(bound, kth_of_lanes(best, a.top));
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const uint64_t k = key(e);
            const bool pass = k <= bound && k != PAD;
            const uint64_t mask = __ballot(pass);
            if (mask == 0) continue;
            if (pass) queue[count + __builtin_popcountll(mask & ((1ull << lane) - 1))] = k;
            count += (uint32_t)__builtin_popcountll(mask);
            if (count > QUEUE - 64) {
                count = shorten(queue, count, a.top, lane);
                if (count == a.top) bound = min(bound, queue[a.top - 1]);
            }
        }
        bound_value = bound == PAD ? -__builtin_inff() : value_of(bound);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
        s = joined(s, {__shfl_xor(s.m, off, 64), __shfl_xor(s.z, off, 64), __shfl_xor(s.t, off, 64)});
    if (lane == 0) wave_stats[wave] = s, wave_bound[wave] = bound, wave_count[wave] = count;
    if (tid == 0) listed = 0;
    __syncthreads();
    s = wave_stats[0];
    bound = wave_bound[0];
#pragma unroll
    for (uint32_t w = 1; w < WAVES; ++w) s = joined(s, wave_stats[w]), bound = min(bound, wave_bound[w]);
    for (uint32_t i = tid; i < WAVES * QUEUE; i += THREADS)
        if (i % QUEUE < wave_count[i / QUEUE] && queues[i / QUEUE][i % QUEUE] <= bound)
            list[atomicAdd(&listed, 1u)] = queues[i / QUEUE][i % QUEUE];
    __syncthreads();
    const uint32_t n = listed;
    if (a.splits == 1) {
        finish<T>(a, row, s, list, n, tid);
        return;
    }
    if (tid == 0) {
        float *to = a.stats + 3 * (uint64_t)blockIdx.x;
        to[0] = s.m, to[1] = s.z, to[2] = s.t;
    }
    uint64_t *to = a.keys + (uint64_t)blockIdx.x * a.top;
    for (uint32_t i = tid; i < n; i += THREADS) {
        const uint64_t mine = list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += list[j] < mine;
        if (rank < a.top) to[rank] = mine;
    }
    for (uint32_t i = n + tid; i < a.top; i += THREADS) to[i] = PAD;
}

// Joins a row's splits (at most 64): their statistics in order, and of their
// sorted keys those that can be among the k best. With the c-th key of every
// split, c = ceil(k / splits): where c is 1, the k-th best of the first keys
// bounds the answer, otherwise the worst of the c-th ones does.
template <typename T> __global__ void __launch_bounds__(THREADS) logprobs_join_kernel(LogprobArgs a) {
    __shared__ uint64_t list[64 * 32];
    __shared__ uint64_t shared_bound;
    __shared__ uint32_t listed;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const float *stats = a.stats + 3 * (uint64_t)row * a.splits;
    const uint64_t *keys = a.keys + (uint64_t)row * a.splits * a.top;
    Stats s = {LOWEST, 0.0f, 0.0f};
    if (lane < a.splits) s = {stats[3 * lane], stats[3 * lane + 1], stats[3 * lane + 2]};
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
        s = joined(s, {__shfl_xor(s.m, off, 64), __shfl_xor(s.z, off, 64), __shfl_xor(s.t, off, 64)});
    if (tid == 0) listed = 0;
    if (tid < 64 && a.top) {
        const uint32_t c = (a.top + a.splits - 1) / a.splits;
        uint64_t key = lane < a.splits ? keys[lane * a.top + c - 1] : c == 1 ? PAD : 0;
        if (c == 1) {
            key = kth_of_lanes(key, a.top);
        } else {
            for (int off = 32; off > 0; off >>= 1)
                key = max(key, (uint64_t)__shfl_xor((unsigned long long)key, off, 64));
        }
        if (lane == 0) shared_bound = key;
    }
    __syncthreads();
    for (uint32_t i = tid; i < a.splits * a.top; i += THREADS) {
        const uint64_t key = keys[i];
        if (key <= shared_bound && key != PAD) list[atomicAdd(&listed, 1u)] = key;
    }
    __syncthreads();
    finish<T>(a, row, s, list, listed, tid);
}

uint32_t splits_of(uint32_t rows, uint32_t count) {
    // one step of a workgroup is 4096 logits; four workgroups a CU fill the card
    const uint32_t steps = (count + THREADS * EACH - 1) / (THREADS * EACH);
    const uint32_t wanted = (1024 + rows - 1) / rows;
    return wanted < steps ? (wanted < 64 ? wanted : 64) : (steps < 64 ? steps : 64);
}

}  // namespace

uint64_t logprobs_floats(uint32_t rows, uint32_t count, uint32_t top) {
    const uint64_t splits = splits_of(rows, count);
    return splits == 1 ? 0 : rows * splits * (2ull * top + 3);
}

hipError_t launch_logprobs(hipStream_t s, const void *logits, uint32_t f16, uint32_t rows, uint32_t count,
                           uint64_t stride, const int32_t *targets, uint32_t top, float *logprobs, float *entropy,
                           uint32_t *ids, float *tops, float *work, uint64_t floats) {
    LogprobArgs a = {logits, stride, targets, logprobs, entropy, ids, tops, rows, count, top, 1, 0, nullptr, nullptr};
    a.splits = splits_of(rows, count);
    if (a.splits > 1 && logprobs_floats(rows, count, top) > floats) a.splits = 1;
    const uint32_t v = f16 ? 8 : 4, step = THREADS * EACH / v;
    const uint64_t vectors = ((uint64_t)count + v - 1 + v - 1) / v;  // a row may begin inside a vector
    a.span = (uint32_t)((vectors + a.splits - 1) / a.splits + step - 1) / step * step;
    a.splits = (uint32_t)((vectors + a.span - 1) / a.span);
    a.keys = (uint64_t *)work;
    a.stats = work + 2ull * rows * a.splits * top;
    if (f16) logprobs_kernel<_Float16><<<rows * a.splits, THREADS, 0, s>>>(a);
    else logprobs_kernel<float><<<rows * a.splits, THREADS, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    if (f16) logprobs_join_kernel<_Float16><<<rows, THREADS, 0, s>>>(a);
    else logprobs_join_kernel<float><<<rows, THREADS, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace nuq
