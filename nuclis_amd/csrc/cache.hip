// Writing tokens into the quantised K/V cache and reading them back (layout
// and formulas: cache.h).
//
// Both kernels give one lane the same 8 consecutive dimensions of a token's K
// and of its V: 16 or 32 bytes of values each, one or two words of codes each.
// A group's extremes are a reduction over the 4 lanes that hold it; a
// non-finite value anywhere in the token-head is a vote over its D / 8 lanes.
// Four tokens in order share a wave at D = 128, so tokens in consecutive slots
// fill whole 256-byte runs of both planes. Memory bound: per token-head 2 D
// values on one side and D (4 bits + 2) / 16 bytes on the other.
#include "cache.h"
#include "kernels.h"

namespace nuq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

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

template <typename T> __device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        half8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];  // exact: the cache's values are f16 numbers
        *(half8 *)p = h;
    } else {
        ((float4 *)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4 *)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

__device__ __forceinline__ float bf16_round(float x) {  // finite x, to nearest even
    uint32_t u = __float_as_uint(x);
    u += 0x7fffu + ((u >> 16) & 1u);
    return __uint_as_float(u & 0xffff0000u);
}

// The scale of the 32-value group that this lane and its 3 neighbours hold.
template <int BITS> __device__ __forceinline__ _Float16 group_scale(const float (&x)[8]) {
    float high = x[0], low = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) high = fmaxf(high, x[i]), low = fminf(low, x[i]);
    high = fmaxf(high, __shfl_xor(high, 1, 64)), low = fminf(low, __shfl_xor(low, 1, 64));
    high = fmaxf(high, __shfl_xor(high, 2, 64)), low = fminf(low, __shfl_xor(low, 2, 64));
    if constexpr (BITS == 4) {
        const float m = high >= -low ? high : low;
        return (_Float16)bf16_round(fminf(fmaxf(m * -0.125f, -2720.0f), 2720.0f));
    } else {
        const uint32_t u = __float_as_uint(fmaxf(high, -low) / 127.0f);
        return (_Float16)fminf(__uint_as_float((u + 0xfffffu) & ~0xfffffu), 56.0f);
    }
}

// Codes with their offset. The division is IEEE's, so a code is the nearest one.
template <int BITS> __device__ __forceinline__ void encode(const float (&x)[8], float d, uint32_t (&q)[8]) {
    constexpr float LOW = BITS == 4 ? -8.0f : -127.0f, HIGH = BITS == 4 ? 7.0f : 127.0f;
    constexpr int OFFSET = BITS == 4 ? 8 : 128;
    const float by = d == 0.0f ? 1.0f : d;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = fminf(fmaxf(rintf(x[i] / by), LOW), HIGH);
        q[i] = d == 0.0f ? (uint32_t)OFFSET : (uint32_t)((int)c + OFFSET);
    }
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
    const uint32_t head = blockIdx.y;
    const uint64_t t = (uint64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    uint8_t *tile = nullptr;
    int n = 0;
    const bool live = t < tokens && locate<BITS, D>(c, slots[t < tokens ? t : 0], head, tile, n);
    float xk[8] = {}, xv[8] = {};
    if (live) {
        load8(k + t * k_stride + head * D + 8 * i, xk);
        load8(v + t * v_stride + head * D + 8 * i, xv);
    }
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) bad |= !isfinite(xk[e]) || !isfinite(xv[e]);
    const uint64_t votes = __ballot(bad) >> (lane / LANES * LANES);
    const bool poison = (votes & (LANES == 64 ? ~0ull : (1ull << (LANES & 63)) - 1)) != 0;
    if (poison) {
#pragma unroll
        for (int e = 0; e < 8; ++e) xk[e] = xv[e] = 0.0f;
    }
    const _Float16 dk = group_scale<BITS>(xk), dv = group_scale<BITS>(xv);
    if (!live) return;
    uint32_t q[8];
    encode<BITS>(xk, (float)dk, q);
    if constexpr (BITS == 4) {
        uint32_t w = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) w |= q[2 * p] << (4 * p) | q[2 * p + 1] << (16 + 4 * p);
        *(uint32_t *)(tile + P::k_codes(n, i)) = w;
    } else {
        *(uint2 *)(tile + P::k_codes(n, i)) = make_uint2(q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24,
                                                         q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24);
    }
    encode<BITS>(xv, (float)dv, q);
    uint8_t *pv = tile + P::v_codes(n, i);
    if constexpr (BITS == 4 && G::COLUMN == 8) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= q[j] << (4 * j);
        *(uint32_t *)pv = w;
    } else if constexpr (BITS == 4) {
        *(uint16_t *)pv = (uint16_t)(q[0] | q[1] << 4 | q[2] << 8 | q[3] << 12);
        *(uint16_t *)(pv + P::V_STEP) = (uint16_t)(q[4] | q[5] << 4 | q[6] << 8 | q[7] << 12);
    } else {
        *(uint32_t *)pv = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
        *(uint32_t *)(pv + P::V_STEP) = q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24;
    }
    if ((i & 3) == 0) {
        *(_Float16 *)(tile + P::k_scale(n, i)) = poison ? (_Float16)__builtin_nanf("") : dk;
        *(_Float16 *)(tile + P::v_scale(n, i)) = dv;
    }
}

template <int BITS, int D, typename T>
__global__ void __launch_bounds__(256) cache_read_kernel(CacheView c, const int64_t *__restrict__ slots,
                                                         uint64_t tokens, T *__restrict__ k, T *__restrict__ v,
                                                         uint64_t k_stride, uint64_t v_stride) {
    using G = CacheGeometry<BITS, D>;
    using P = Place<BITS, D>;
    constexpr int LANES = D / 8;
    const int i = (int)(threadIdx.x % LANES);
    const uint32_t head = blockIdx.y;
    const uint64_t t = (uint64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (t >= tokens) return;
    uint8_t *tile;
    int n;
    float xk[8] = {}, xv[8] = {};  // no such slot: zeros
    if (locate<BITS, D>(c, slots[t], head, tile, n)) {
        const float dk = (float)*(const _Float16 *)(tile + P::k_scale(n, i));
        float dv = (float)*(const _Float16 *)(tile + P::v_scale(n, i));
        if (dk != dk) dv = dk;  // a token-head that held a non-finite value
        const uint8_t *pk = tile + P::k_codes(n, i), *pv = tile + P::v_codes(n, i);
        if constexpr (BITS == 4) {
            const uint32_t a = *(const uint32_t *)pk;
            uint32_t b;
            if constexpr (G::COLUMN == 8) b = *(const uint32_t *)pv;
            else b = *(const uint16_t *)pv | (uint32_t)*(const uint16_t *)(pv + P::V_STEP) << 16;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xk[e] = (float)((int)(a >> (4 * (e >> 1) + 16 * (e & 1)) & 15u) - G::OFFSET) * dk;
                xv[e] = (float)((int)(b >> (4 * e) & 15u) - G::OFFSET) * dv;
            }
        } else {
            const uint2 a = *(const uint2 *)pk;
            const uint32_t b[2] = {*(const uint32_t *)pv, *(const uint32_t *)(pv + P::V_STEP)};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xk[e] = (float)((int)((e < 4 ? a.x : a.y) >> (8 * (e & 3)) & 255u) - G::OFFSET) * dk;
                xv[e] = (float)((int)(b[e >> 2] >> (8 * (e & 3)) & 255u) - G::OFFSET) * dv;
            }
        }
    }
    store8(k + t * k_stride + head * D + 8 * i, xk);
    store8(v + t * v_stride + head * D + 8 * i, xv);
}

template <int BITS, int D>
hipError_t write_d(hipStream_t s, const CacheView &c, uint32_t f16, const void *k, const void *v, uint64_t k_stride,
                   uint64_t v_stride, const int64_t *slots, uint64_t tokens) {
    const dim3 grid((uint32_t)((tokens + 2048 / D - 1) / (2048 / D)), c.kv_heads);
    if (f16)
        cache_write_kernel<BITS, D><<<grid, 256, 0, s>>>(c, (const _Float16 *)k, (const _Float16 *)v, k_stride,
                                                         v_stride, slots, tokens);
    else
        cache_write_kernel<BITS, D><<<grid, 256, 0, s>>>(c, (const float *)k, (const float *)v, k_stride, v_stride,
                                                         slots, tokens);
    return hipGetLastError();
}

template <int BITS, int D>
hipError_t read_d(hipStream_t s, const CacheView &c, uint32_t f16, const int64_t *slots, uint64_t tokens, void *k,
                  void *v, uint64_t k_stride, uint64_t v_stride) {
    const dim3 grid((uint32_t)((tokens + 2048 / D - 1) / (2048 / D)), c.kv_heads);
    if (f16)
        cache_read_kernel<BITS, D><<<grid, 256, 0, s>>>(c, slots, tokens, (_Float16 *)k, (_Float16 *)v, k_stride,
                                                        v_stride);
    else
        cache_read_kernel<BITS, D><<<grid, 256, 0, s>>>(c, slots, tokens, (float *)k, (float *)v, k_stride, v_stride);
    return hipGetLastError();
}

}  // namespace

uint64_t cache_tile_bytes(uint32_t bits, uint32_t head_dim) { return (uint64_t)head_dim * (4 * bits + 2); }

hipError_t launch_cache_write(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f16,
                              const void *k, const void *v, uint64_t k_stride, uint64_t v_stride, const int64_t *slots,
                              uint64_t tokens) {
#define NUQ_CASE(B, D) \
    if (bits == B && head_dim == D) return write_d<B, D>(s, c, f16, k, v, k_stride, v_stride, slots, tokens);
    NUQ_CASE(4, 64) NUQ_CASE(4, 128) NUQ_CASE(4, 256) NUQ_CASE(8, 64) NUQ_CASE(8, 128) NUQ_CASE(8, 256)
#undef NUQ_CASE
    return hipErrorInvalidValue;
}

hipError_t launch_cache_read(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f16,
                             const int64_t *slots, uint64_t tokens, void *k, void *v, uint64_t k_stride,
                             uint64_t v_stride) {
#define NUQ_CASE(B, D) \
    if (bits == B && head_dim == D) return read_d<B, D>(s, c, f16, slots, tokens, k, v, k_stride, v_stride);
    NUQ_CASE(4, 64) NUQ_CASE(4, 128) NUQ_CASE(4, 256) NUQ_CASE(8, 64) NUQ_CASE(8, 128) NUQ_CASE(8, 256)
#undef NUQ_CASE
    return hipErrorInvalidValue;
}

}  // namespace nuq
