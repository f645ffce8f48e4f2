// Writing tokens into the quantised K/V cache and reading them back (layout
// and formulas: cache.h).
//
// Writing. One lane holds 8 consecutive dimensions of a token's K and of its V: 16
// or 32 bytes of values each, one or two words of codes each. A group's extremes
// are a reduction over the 4 lanes that hold it; a non-finite value anywhere in
// the token-head is a vote over its D / 8 lanes. Tokens in order share a wave (four
// at D = 128), so tokens in consecutive slots fill whole 256-byte runs of both planes.
//
// Memory bound: per token-head 2 D values on one side and D (4 bits + 2) / 16 bytes on
// the other. The heads of a token are neighbours in the grid, as their values are in
// memory. Read values go out past the caches in whole lines. 32768 tokens of 8 heads of
// 128, 4 bits: F16 25 us, 6.8 TB/s, F32 46 us, 6.6 TB/s (8 bits 30 and 50 us). Calls right
// behind each other: F16 29 us, 41 with ordinary stores, F32 47 and 75; with a product that
// reads the values behind each, F16 75 and 70 (so much of it comes back there), F32 140 and
// 151. Writing the same takes 38 us (4.5 TB/s) and 58 us (5.3), at 8 bits 45 and 65: about 300
// vector instructions a wave of 512 values of each plane, as long as the memory takes.
#include "cache.h"
#include "kernels.h"

#include <algorithm>

namespace nuq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        const half8 h = *(const half8 *)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    } else {
        const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
}

__device__ __forceinline__ float bf16_round(float x) {  // finite x, to nearest even
    uint32_t u = __float_as_uint(x);
    u += 0x7fffu + ((u >> 16) & 1u);
    return __uint_as_float(u & 0xffff0000u);
}

// The value of the lane at `quad_perm` CONTROL in its group of four.
template <int CONTROL> __device__ __forceinline__ float in_quad(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CONTROL, 0xf, 0xf, true));
}

// The scale of the 32-value group that this lane and its 3 neighbours hold, and its largest magnitude.
template <int BITS> __device__ __forceinline__ _Float16 group_scale(const float (&x)[8], float &most) {
    float high = x[0], low = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) high = fmaxf(high, x[i]), low = fminf(low, x[i]);
    high = fmaxf(high, in_quad<0xb1>(high)), low = fminf(low, in_quad<0xb1>(low));  // lane ^ 1
    high = fmaxf(high, in_quad<0x4e>(high)), low = fminf(low, in_quad<0x4e>(low));  // lane ^ 2
    most = fmaxf(high, -low);
    if constexpr (BITS == 4) {
        const float m = high >= -low ? high : low;
        return (_Float16)bf16_round(fminf(fmaxf(m * -0.125f, -2720.0f), 2720.0f));
    } else {
        const uint32_t u = __float_as_uint(most / 127.0f);
        return (_Float16)fminf(__uint_as_float((u + 0xfffffu) & ~0xfffffu), 56.0f);
    }
}

// Codes with their offset, as the low bits of a word whose others are MAGIC's: the
// nearest code to x / d as IEEE divides. Its quotients come from the group's
// reciprocal r, rounded to nearest, and two steps (Markstein 1990): q0 = x r, then
// q0 + (x - q0 d) r with the residual exact. Where a group holds more than a code can
// reach, inputs are clamped first (d <= 2720, so 1e6 / d saturates either range),
// which keeps the residual finite. A group of d = 0 holds numbers that round to 0.
// Adding 2^23 rounds to an integer, ties to even, and leaves it in the low bits.
constexpr uint32_t MAGIC = 0x4b000000u;  // of 2^23
template <int BITS> __device__ __forceinline__ void encode(float (&x)[8], float d, float most, uint32_t (&q)[8]) {
    constexpr float LOW = BITS == 4 ? -8.0f : -127.0f, HIGH = BITS == 4 ? 7.0f : 127.0f;
    constexpr float OFFSET = BITS == 4 ? 8.0f : 128.0f;
    const float by = d == 0.0f ? 1.0f : d, r = 1.0f / by;
    if (__any(most > 1e6f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_fmed3f(x[i], -1e6f, 1e6f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q0 = x[i] * r, c = fmaf(fmaf(-q0, by, x[i]), r, q0);
        q[i] = __float_as_uint(__builtin_amdgcn_fmed3f(c, LOW, HIGH) + (8388608.0f + OFFSET));
    }
}
// Codes q[0..N) side by side, the i-th at bit shift(i); MAGIC's bits fall out of the sum.
template <int N, typename Shift> __device__ __forceinline__ uint32_t packed(const uint32_t *q, Shift shift) {
    uint32_t w = 0, magic = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) w = (q[i] << shift(i)) + w, magic += MAGIC << shift(i);
    return w - magic;
}

template <int BITS, int D> struct Place {
    using G = CacheGeometry<BITS, D>;
    // The lane's dimensions are 8 i ..+7 of token n of the tile.
    static __device__ __forceinline__ uint32_t k_codes(int n, int i) {
        const int g = i >> 2, u = g / G::UNIT_GROUPS;
        return ((u * 16 + n) * 4 + (i & 3)) * G::CHUNK + (g % G::UNIT_GROUPS) * BITS;
    }
    static __device__ __forceinline__ uint32_t k_scale(int n, int i) {
        return G::K_SCALES + 2 * (n * G::GROUPS + (i >> 2));
    }
    // first of the 8 / COLUMN columns the lane's dimensions fill
    static __device__ __forceinline__ uint32_t v_codes(int n, int i) {
        const int u = 8 * i / G::UNIT_DIMS, column = 8 * i % G::UNIT_DIMS / G::COLUMN;
        return G::V_CODES + (((u * 4 + (n >> 2)) * 16 + column) * 4 + (n & 3)) * (G::CHUNK / 4);
    }
    static constexpr uint32_t V_STEP = G::CHUNK;  // bytes from a column to the next
    static __device__ __forceinline__ uint32_t v_scale(int n, int i) {
        return G::V_SCALES + 2 * (((n >> 2) * G::GROUPS + (i >> 2)) * 4 + (n & 3));
    }
};

// Where token `slot` of head `head` lives; false where there is no such slot.
template <int BITS, int D>
__device__ __forceinline__ bool locate(const CacheView &c, int64_t slot, uint32_t head, uint8_t *&tile, int &n) {
    const uint64_t at = (uint64_t)slot >> 4, page = at >> c.tiles_log2;
    if (slot < 0 || page >= c.pages) return false;
    const uint64_t in_page = at & ((1ull << c.tiles_log2) - 1);
    tile = c.bytes + (((page * c.kv_heads + head) << c.tiles_log2) + in_page) * CacheGeometry<BITS, D>::TILE_BYTES;
    n = (int)(slot & 15);
    return true;
}

template <int BITS, int D, typename T>
__global__ void __launch_bounds__(256) cache_write_kernel(CacheView c, const T *__restrict__ k, const T *__restrict__ v,
                                                          uint64_t k_stride, uint64_t v_stride,
                                                          const int64_t *__restrict__ slots, uint64_t tokens) {
    using G = CacheGeometry<BITS, D>;
    using P = Place<BITS, D>;
    constexpr int LANES = D / 8;  // of a token-head
    const uint32_t lane = threadIdx.x & 63;
    const int i = (int)(threadIdx.x % LANES);
    const uint32_t head = blockIdx.x % c.kv_heads;
    const uint64_t t = (uint64_t)(blockIdx.x / c.kv_heads) * (256 / LANES) + threadIdx.x / LANES;
    uint8_t *tile = nullptr;
    int n = 0;
    // (values and slot are on the way together: a token without a slot is read and not written)
    const uint64_t from = t < tokens ? t : tokens - 1;
    float xk[8], xv[8];
    load8(k + from * k_stride + head * D + 8 * i, xk);
    load8(v + from * v_stride + head * D + 8 * i, xv);
    const bool live = locate<BITS, D>(c, slots[from], head, tile, n) && t < tokens;
    float finite = 0.0f;  // 0 x is NaN where x is not finite
#pragma unroll
    for (int e = 0; e < 8; ++e) finite = fmaf(xk[e], 0.0f, finite), finite = fmaf(xv[e], 0.0f, finite);
    const uint64_t bad = __ballot(finite != finite), votes = bad >> (lane / LANES * LANES);
    const bool poison = (votes & (LANES == 64 ? ~0ull : (1ull << (LANES & 63)) - 1)) != 0;
    if (bad) {
#pragma unroll
        for (int e = 0; e < 8; ++e) xk[e] = poison ? 0.0f : xk[e], xv[e] = poison ? 0.0f : xv[e];
    }
    float most_k, most_v;
    const _Float16 dk = group_scale<BITS>(xk, most_k), dv = group_scale<BITS>(xv, most_v);
    uint32_t q[8];
    encode<BITS>(xk, (float)dk, most_k, q);
    uint32_t k_words[2], v_words[2];
    const auto bytes = [](int e) { return 8 * e; };
    const auto nibbles = [](int e) { return 4 * e; };
    if constexpr (BITS == 4) k_words[0] = packed<8>(q, [](int e) { return 4 * (e >> 1) + 16 * (e & 1); });
    else k_words[0] = packed<4>(q, bytes), k_words[1] = packed<4>(q + 4, bytes);
    encode<BITS>(xv, (float)dv, most_v, q);
    if constexpr (BITS == 4 && G::COLUMN == 8) v_words[0] = packed<8>(q, nibbles);
    else if constexpr (BITS == 4) v_words[0] = packed<4>(q, nibbles), v_words[1] = packed<4>(q + 4, nibbles);
    else v_words[0] = packed<4>(q, bytes), v_words[1] = packed<4>(q + 4, bytes);
    if (!live) return;
    uint8_t *pk = tile + P::k_codes(n, i), *pv = tile + P::v_codes(n, i);
    if constexpr (BITS == 4) {
        *(uint32_t *)pk = k_words[0];
        if constexpr (G::COLUMN == 8) *(uint32_t *)pv = v_words[0];
        else *(uint16_t *)pv = (uint16_t)v_words[0], *(uint16_t *)(pv + P::V_STEP) = (uint16_t)v_words[1];
    } else {
        *(uint2 *)pk = make_uint2(k_words[0], k_words[1]);
        *(uint32_t *)pv = v_words[0], *(uint32_t *)(pv + P::V_STEP) = v_words[1];
    }
    if ((i & 3) == 0) {
        *(_Float16 *)(tile + P::k_scale(n, i)) = poison ? (_Float16)__builtin_nanf("") : dk;
        *(_Float16 *)(tile + P::v_scale(n, i)) = dv;
    }
}

// The 4 codes, as they stand with their offset, of dimensions 4 * quad ..+3 of token n.
template <int BITS, int D>
__device__ __forceinline__ void k_quad(const uint8_t *tile, int n, int quad, uint32_t (&q)[4]) {
    const uint8_t *p = tile + Place<BITS, D>::k_codes(n, quad >> 1);
    const uint32_t w = *(const uint32_t *)(BITS == 4 ? p : p + 4 * (quad & 1)), by = BITS == 4 ? 8 * (quad & 1) : 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        q[e] = BITS == 4 ? w >> (by + 4 * (e >> 1) + 16 * (e & 1)) & 15u : w >> (8 * e) & 255u;
}
template <int BITS, int D>
__device__ __forceinline__ void v_quad(const uint8_t *tile, int n, int quad, uint32_t (&q)[4]) {
    using P = Place<BITS, D>;
    const uint8_t *p = tile + P::v_codes(n, quad >> 1);
    uint32_t w;
    if constexpr (BITS == 8) w = *(const uint32_t *)(p + (quad & 1) * P::V_STEP);
    else if constexpr (CacheGeometry<BITS, D>::COLUMN == 8) w = *(const uint16_t *)(p + 2 * (quad & 1));
    else w = *(const uint16_t *)(p + (quad & 1) * P::V_STEP);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = w >> (BITS * e) & ((1u << BITS) - 1);
}

// A lane takes 16 bytes of each result at a time, so that a wave's store is whole
// lines of them: 4 dimensions, F16 8.
template <int BITS, int D, typename T>
__global__ void __launch_bounds__(256) cache_read_kernel(CacheView c, const int64_t *__restrict__ slots,
                                                         uint64_t tokens, T *__restrict__ k, T *__restrict__ v,
                                                         uint64_t k_stride, uint64_t v_stride) {
    using G = CacheGeometry<BITS, D>;
    using P = Place<BITS, D>;
    typedef T vector __attribute__((ext_vector_type(16 / sizeof(T))));
    // D / 8 lanes hold a token-head: F32 in two passes of 4 dimensions, F16 in one of 8
    constexpr int LANES = D / 8, QUADS = sizeof(T) == 2 ? 2 : 1, PASSES = sizeof(T) / 2;
    const uint32_t head = blockIdx.x % c.kv_heads;
    const uint64_t t = (uint64_t)(blockIdx.x / c.kv_heads) * (256 / LANES) + threadIdx.x / LANES;
    if (t >= tokens) return;
    uint8_t *tile = c.bytes;  // no such slot: the cache's first token is read and zeros are written
    int n = 0;
    const bool live = locate<BITS, D>(c, slots[t], head, tile, n);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        const int at = (int)(threadIdx.x % LANES) + pass * LANES;
        vector xk, xv;
        const float dk = (float)*(const _Float16 *)(tile + P::k_scale(n, at * QUADS / 2));
        float dv = (float)*(const _Float16 *)(tile + P::v_scale(n, at * QUADS / 2));
        if (dk != dk) dv = dk;  // a token-head that held a non-finite value
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            uint32_t q[4];
            k_quad<BITS, D>(tile, n, at * QUADS + j, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) xk[4 * j + e] = live ? (T)((float)((int)q[e] - G::OFFSET) * dk) : (T)0.0f;
            v_quad<BITS, D>(tile, n, at * QUADS + j, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) xv[4 * j + e] = live ? (T)((float)((int)q[e] - G::OFFSET) * dv) : (T)0.0f;
        }
        const uint64_t to = head * D + at * 4 * QUADS;
        u32x4 wk = __builtin_bit_cast(u32x4, xk), wv = __builtin_bit_cast(u32x4, xv);
        asm volatile("" : "+v"(wk), "+v"(wv));  // (the optimiser otherwise forgets that an F16 store is nontemporal)
        __builtin_nontemporal_store(wk, (u32x4 *)(k + t * k_stride + to));
        __builtin_nontemporal_store(wv, (u32x4 *)(v + t * v_stride + to));
    }
}

// A grid holds less than 2^32 threads: many tokens go in pieces.
template <int D, typename Launch> hipError_t in_pieces(const CacheView &c, uint64_t tokens, Launch launch) {
    constexpr uint64_t EACH = 2048 / D;  // tokens of a workgroup
    const uint64_t most = (((1ull << 23) + c.kv_heads - 1) / c.kv_heads) * EACH;
    for (uint64_t first = 0; first < tokens; first += most) {
        const uint64_t count = std::min(most, tokens - first);
        launch((uint32_t)((count + EACH - 1) / EACH * c.kv_heads), first, count);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int BITS, int D, typename T>
hipError_t write_d(hipStream_t s, const CacheView &c, const T *k, const T *v, uint64_t k_stride, uint64_t v_stride,
                   const int64_t *slots, uint64_t tokens) {
    return in_pieces<D>(c, tokens, [&](uint32_t grid, uint64_t first, uint64_t count) {
        cache_write_kernel<BITS, D><<<grid, 256, 0, s>>>(c, k + first * k_stride, v + first * v_stride, k_stride,
                                                         v_stride, slots + first, count);
    });
}

template <int BITS, int D, typename T>
hipError_t read_d(hipStream_t s, const CacheView &c, const int64_t *slots, uint64_t tokens, T *k, T *v,
                  uint64_t k_stride, uint64_t v_stride) {
    return in_pieces<D>(c, tokens, [&](uint32_t grid, uint64_t first, uint64_t count) {
        cache_read_kernel<BITS, D><<<grid, 256, 0, s>>>(c, slots + first, count, k + first * k_stride,
                                                        v + first * v_stride, k_stride, v_stride);
    });
}

}  // namespace

uint64_t cache_tile_bytes(uint32_t bits, uint32_t head_dim) { return (uint64_t)head_dim * (4 * bits + 2); }

hipError_t launch_cache_write(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f16,
                              const void *k, const void *v, uint64_t k_stride, uint64_t v_stride, const int64_t *slots,
                              uint64_t tokens) {
#define NUQ_CASE(B, D) \
    if (bits == B && head_dim == D)                                                                     \
        return f16 ? write_d<B, D>(s, c, (const _Float16 *)k, (const _Float16 *)v, k_stride, v_stride, slots, tokens) \
                   : write_d<B, D>(s, c, (const float *)k, (const float *)v, k_stride, v_stride, slots, tokens);
    NUQ_CASE(4, 64) NUQ_CASE(4, 128) NUQ_CASE(4, 256) NUQ_CASE(8, 64) NUQ_CASE(8, 128) NUQ_CASE(8, 256)
#undef NUQ_CASE
    return hipErrorInvalidValue;
}

hipError_t launch_cache_read(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f16,
                             const int64_t *slots, uint64_t tokens, void *k, void *v, uint64_t k_stride,
                             uint64_t v_stride) {
#define NUQ_CASE(B, D) \
    if (bits == B && head_dim == D)                                                                     \
        return f16 ? read_d<B, D>(s, c, slots, tokens, (_Float16 *)k, (_Float16 *)v, k_stride, v_stride) \
                   : read_d<B, D>(s, c, slots, tokens, (float *)k, (float *)v, k_stride, v_stride);
    NUQ_CASE(4, 64) NUQ_CASE(4, 128) NUQ_CASE(4, 256) NUQ_CASE(8, 64) NUQ_CASE(8, 128) NUQ_CASE(8, 256)
#undef NUQ_CASE
    return hipErrorInvalidValue;
}

}  // namespace nuq
