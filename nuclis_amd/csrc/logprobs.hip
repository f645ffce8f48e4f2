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
// smaller is better. A workgroup keeps the best value of each lane over its four
// waves; the k-th best of these 64 (k <= 32) is a bound that k different logits
// reach, so only logits that reach it can be among the answer. They go to a queue
// in LDS, which one comparison for 16 logits leaves alone almost always: about
// 64 ln(64 / (64 - k)) logits reach the bound of the data so far. At the end the
// waves' queues, cut by the last bound, are ranked by counting.
//
// Bound by the read of the logits: 1024 rows of 151936 F32 logits with five
// alternatives take 99 us, 6.3 TB/s (without alternatives 97; as F16 64). The
// next step's loads are on the way during a step's work, past the caches (111 us
// with ordinary loads: nothing is read twice). Each wave with a bound of its own
// took half as long again: three times the steps looked at single logits.
// A row is split over workgroups where there are few rows, a step each at the
// least; the splits' results go to the workspace for a second kernel. One row
// takes 11 us with twenty alternatives, 64 rows 22 us: a split has a few steps, and
// its candidates are queued from the first on, before a bound is worth anything; then
// comes the second kernel's 4 us.
#include "kernels.h"

namespace nuq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.44269504088896340736f;
constexpr uint64_t PAD = ~0ull;  // after every key
constexpr uint32_t THREADS = 256, WAVES = 4, QUEUE = 256;
constexpr int EACH = 16;         // logits a thread holds at a time

// values in their order as unsigned numbers
constexpr uint32_t LOWEST_ORDER = 0x007fffffu;  // of -inf
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t order) {
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) {
    const uint32_t order = order_of(v == 0.0f ? 0.0f : v);  // -0 ties with +0
    return v != v ? PAD : (uint64_t)~order << 32 | i;
}
__device__ __forceinline__ float value_of(uint64_t key) { return of_order(~(uint32_t)(key >> 32)); }

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

// At most the k-th best of a wave's 64 values, by their order: the largest number of
// 18 bits that k of them reach, a bit at a time. (The 14 bits left out tell values
// within 1/512 of each other apart; the queue takes the few more that they let in.)
__device__ __forceinline__ uint32_t bound_of_lanes(uint32_t order, uint32_t k) {
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 14; --bit) {
        const uint32_t higher = bound | 1u << bit;
        if ((uint32_t)__builtin_popcountll(__ballot(order >= higher)) >= k) bound = higher;
    }
    return max(bound, LOWEST_ORDER);
}

// How many of a list's n keys come before `key`. The reads of eight keys are on
// the way together; the list is padded to eights.
__device__ __forceinline__ uint32_t rank_in(const uint64_t *list, uint32_t n, uint64_t key) {
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; j += 8) {
        uint64_t other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = list[j + i];
#pragma unroll
        for (int i = 0; i < 8; ++i) rank += other[i] < key;
    }
    return rank;
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

// The target's logit: of no use where there is no such token.
template <typename T> __device__ __forceinline__ float target_of(const LogprobArgs &a, uint32_t row, uint32_t *id) {
    *id = (uint32_t)a.targets[row];
    return (float)((const T *)a.logits)[(uint64_t)row * a.stride + min(*id, a.count - 1)];
}

// The row's answer from its statistics; the tops are `list`'s keys by rank.
__device__ __forceinline__ void finish(const LogprobArgs &a, uint32_t row, uint32_t id, float x, const Stats &s,
                                       const uint64_t *list, uint32_t n, uint32_t tid) {
    const float ln_z = logf(s.z);
    if (tid == 0) {
        // a row of -inf alone has no distribution: -inf and no entropy
        const float lp = s.z == 0.0f ? -__builtin_inff() : (x - s.m) - ln_z;
        a.logprobs[row] = id < a.count ? lp : __builtin_nanf("");
        a.entropy[row] = s.z == 0.0f ? 0.0f : ln_z - s.t / s.z;
    }
    for (uint32_t i = tid; i < n; i += THREADS) {
        const uint64_t mine = list[i];
        const uint32_t rank = rank_in(list, n, mine);
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
    __shared__ uint64_t queues[WAVES][QUEUE], list[WAVES * QUEUE + 8];
    __shared__ Stats wave_stats[WAVES];
    __shared__ uint64_t wave_bound[WAVES];
    __shared__ uint32_t wave_count[WAVES], listed, lanes_best[64], shared_bound;
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const T *x = (const T *)a.logits + (uint64_t)row * a.stride;
    // vectors are 16-byte aligned: the first may begin before the row
    const int before = (int)(((uintptr_t)x & 15) / sizeof(T));
    const uint32_t vectors = (uint32_t)((before + (uint64_t)a.count + V - 1) / V);
    const uint32_t end = min(vectors, (split + 1) * a.span);
    uint64_t *queue = queues[wave];
    if (tid < 64) lanes_best[tid] = LOWEST_ORDER;
    if (tid == 64) shared_bound = LOWEST_ORDER, listed = 0;
    uint32_t id = 0;
    float target = 0.0f;
    if (a.splits == 1) target = target_of<T>(a, row, &id);

    Stats s = {LOWEST, 0.0f, 0.0f};
    uint64_t bound = PAD;  // of keys, once a queue has been shortened
    float best = -__builtin_inff();
    uint32_t count = 0;
    // vectors [full, full_end) lie in the row whole
    const uint32_t full = before ? 1 : 0, full_end = (uint32_t)((before + (uint64_t)a.count) / V);
    // The next step's vectors are requested before this step's are worked on, from a
    // whole vector's place whatever theirs: no condition stands between the loads.
    u32x4 next[VECTORS] = {};
    const auto request = [&](uint32_t base) {
#pragma unroll
        for (int u = 0; u < VECTORS; ++u) {
            const uint32_t at = min(max(base + u * THREADS + tid, full), full_end - 1);
            next[u] = __builtin_nontemporal_load(
                (const u32x4 *)((const uint8_t *)x - before * (int)sizeof(T) + 16ull * at));
        }
    };
    if (full < full_end) request(split * a.span);
    __syncthreads();
    for (uint32_t base = split * a.span; base < end; base += THREADS * VECTORS) {
        float v[EACH];
#pragma unroll
        for (int u = 0; u < VECTORS; ++u) {
            if constexpr (V == 4) {
                v[4 * u] = __uint_as_float(next[u].x), v[4 * u + 1] = __uint_as_float(next[u].y);
                v[4 * u + 2] = __uint_as_float(next[u].z), v[4 * u + 3] = __uint_as_float(next[u].w);
            } else {
                const half8 f = __builtin_bit_cast(half8, next[u]);
#pragma unroll
                for (int e = 0; e < V; ++e) v[V * u + e] = (float)f[e];
            }
        }
        if (full < full_end) request(min(base + THREADS * VECTORS, vectors));
        if (base < full || base + THREADS * VECTORS > min(full_end, end)) {  // the row's or the split's edge
#pragma unroll
            for (int u = 0; u < VECTORS; ++u) {
                const uint32_t at = base + u * THREADS + tid;
                if (at >= full && at < full_end && at < end) continue;
                const int64_t first = (int64_t)at * V - before;
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
        // (the waves raise the bound as they come: an older one lets more through, no less)
        uint32_t reach = a.top ? *(volatile uint32_t *)&shared_bound : 0;
        if (a.top == 0 || !__any(most >= of_order(reach))) continue;
        best = fmaxf(best, most);
        atomicMax(&lanes_best[lane], order_of(best));
        reach = max(reach, bound_of_lanes(*(volatile uint32_t *)&lanes_best[lane], a.top));
        if (lane == 0) atomicMax(&shared_bound, reach);
        const float least = of_order((uint32_t)__builtin_amdgcn_readfirstlane((int)reach));
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            if (!__any(v[e] >= least)) continue;
            // absent places (before and behind the row) have no key
            const uint32_t vector = base + e / V * THREADS + tid, i = vector * V - before + e % V;
            const uint64_t k = vector < end && i < a.count ? key_of(v[e], i) : PAD;
            const bool pass = v[e] >= least && k <= bound && k != PAD;
            const uint64_t mask = __ballot(pass);
            if (mask == 0) continue;
            if (pass) queue[count + __builtin_popcountll(mask & ((1ull << lane) - 1))] = k;
            count += (uint32_t)__builtin_popcountll(mask);
            if (count > QUEUE - 64) {
                count = shorten(queue, count, a.top, lane);
                if (count == a.top) bound = min(bound, queue[a.top - 1]);
            }
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
        s = joined(s, {__shfl_xor(s.m, off, 64), __shfl_xor(s.z, off, 64), __shfl_xor(s.t, off, 64)});
    if (lane == 0) wave_stats[wave] = s, wave_bound[wave] = bound, wave_count[wave] = count;
    __syncthreads();
    s = wave_stats[0];
    bound = wave_bound[0];
#pragma unroll
    for (uint32_t w = 1; w < WAVES; ++w) s = joined(s, wave_stats[w]), bound = min(bound, wave_bound[w]);
    // of the keys of one value the bound keeps all
    const uint64_t worst = key_of(of_order(shared_bound), ~0u);
    bound = min(bound, worst);
    for (uint32_t i = tid; i < WAVES * QUEUE; i += THREADS)
        if (i % QUEUE < wave_count[i / QUEUE] && queues[i / QUEUE][i % QUEUE] <= bound)
            list[atomicAdd(&listed, 1u)] = queues[i / QUEUE][i % QUEUE];
    __syncthreads();
    const uint32_t n = listed;
    if (tid < 8) list[n + tid] = PAD;
    __syncthreads();
    if (a.splits == 1) {
        finish(a, row, id, target, s, list, n, tid);
        return;
    }
    if (tid == 0) {
        float *to = a.stats + 3 * (uint64_t)blockIdx.x;
        to[0] = s.m, to[1] = s.z, to[2] = s.t;
    }
    uint64_t *to = a.keys + (uint64_t)blockIdx.x * a.top;
    for (uint32_t i = tid; i < n; i += THREADS) {
        const uint64_t mine = list[i];
        const uint32_t rank = rank_in(list, n, mine);
        if (rank < a.top) to[rank] = mine;
    }
    for (uint32_t i = n + tid; i < a.top; i += THREADS) to[i] = PAD;
}

// Joins a row's splits (at most 64): their statistics in order, and of their
// sorted keys those that can be among the k best. With the c-th key of every
// split, c = ceil(k / splits): where c is 1, the k-th best of the first keys
// bounds the answer, otherwise the worst of the c-th ones does.
template <typename T> __global__ void __launch_bounds__(THREADS) logprobs_join_kernel(LogprobArgs a) {
    __shared__ uint64_t list[64 * 32 + 8];
    __shared__ uint64_t shared_bound;
    __shared__ uint32_t listed;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const float *stats = a.stats + 3 * (uint64_t)row * a.splits;
    const uint64_t *keys = a.keys + (uint64_t)row * a.splits * a.top;
    constexpr int HELD = 64 * 32 / THREADS;
    uint64_t held[HELD];  // every load on the way before the first is waited for
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = tid + THREADS * i < a.splits * a.top ? keys[tid + THREADS * i] : PAD;
    uint32_t id;
    const float target = target_of<T>(a, row, &id);
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
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (held[i] <= shared_bound && held[i] != PAD) list[atomicAdd(&listed, 1u)] = held[i];
    __syncthreads();
    const uint32_t n = listed;
    if (tid < 8) list[n + tid] = PAD;
    __syncthreads();
    finish(a, row, id, target, s, list, n, tid);
}

uint32_t splits_of(uint32_t rows, uint32_t count, uint32_t cus) {
    // one step of a workgroup is 4096 logits; four workgroups a CU fill the card
    const uint32_t steps = (count + THREADS * EACH - 1) / (THREADS * EACH);
    const uint32_t wanted = (4 * cus + rows - 1) / rows;
    return wanted < steps ? (wanted < 64 ? wanted : 64) : (steps < 64 ? steps : 64);
}

}  // namespace

uint64_t logprobs_floats(uint32_t rows, uint32_t count, uint32_t top, uint32_t cus) {
    const uint64_t splits = splits_of(rows, count, cus);
    return splits == 1 ? 0 : rows * splits * (2ull * top + 3);
}

hipError_t launch_logprobs(hipStream_t s, const void *logits, uint32_t f16, uint32_t rows, uint32_t count,
                           uint64_t stride, const int32_t *targets, uint32_t top, float *logprobs, float *entropy,
                           uint32_t *ids, float *tops, float *work, uint64_t floats, uint32_t cus) {
    LogprobArgs a = {logits, stride, targets, logprobs, entropy, ids, tops, rows, count, top, 1, 0, nullptr, nullptr};
    a.splits = splits_of(rows, count, cus);
    if (a.splits > 1 && logprobs_floats(rows, count, top, cus) > floats) a.splits = 1;
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
