// What the attention kernels share: the cache's tiles as matrix operands, and the
// rows and steps a workgroup works on (attention.hip, attention_prompt.hip).
#pragma once

#include "attention.h"

namespace nuq {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float LOWEST = -3.402823466e38f;  // a running maximum before any token
constexpr float RAISE = 7.0f;   // P is 2^RAISE at the reference
constexpr float SLACK = 8.0f;   // how far (log2) a score may pass the reference
constexpr int WAVES = 4, MAX_SPLITS = 64;

__device__ __forceinline__ half2v as_half2(uint32_t u) { return __builtin_bit_cast(half2v, u); }
__device__ __forceinline__ uint32_t as_u32(half2v h) { return __builtin_bit_cast(uint32_t, h); }

struct Operand {  // 8 f16 of one lane
    uint32_t w[4];
    __device__ __forceinline__ half8 get() const { return __builtin_bit_cast(half8, *this); }
};

// A nibble in the top mantissa bits of 16.0 is 16 + code; a byte under 0x64 is
// 1024 + code. One f16 fma by (d, -bias d) then gives d * (code - offset) exactly.
template <int BITS> __device__ __forceinline__ half2v bias_of(half2v d) {
    return d * (_Float16)(BITS == 4 ? -24.0f : -1152.0f);
}
// The pair of nibbles at bits p and 16 + p, p = 4 I.
template <int I> __device__ __forceinline__ uint32_t nibbles(uint32_t w) {
    constexpr int SHIFT = 6 - 4 * I;
    const uint32_t s = SHIFT >= 0 ? w << (SHIFT >= 0 ? SHIFT : 0) : w >> (SHIFT >= 0 ? 0 : -SHIFT);
    return (s & 0x03c003c0u) | 0x4c004c00u;
}

// 8 dimensions of one token.
__device__ __forceinline__ Operand decode_k4(uint32_t w, half2v d, half2v b) {
    return {{as_u32(as_half2(nibbles<0>(w)) * d + b), as_u32(as_half2(nibbles<1>(w)) * d + b),
             as_u32(as_half2(nibbles<2>(w)) * d + b), as_u32(as_half2(nibbles<3>(w)) * d + b)}};
}
__device__ __forceinline__ Operand decode_k8(uint32_t w0, uint32_t w1, half2v d, half2v b) {
    constexpr uint32_t HIGH = 0x64646464u;
    return {{as_u32(as_half2(__builtin_amdgcn_perm(HIGH, w0, 0x04010400u)) * d + b),
             as_u32(as_half2(__builtin_amdgcn_perm(HIGH, w0, 0x04030402u)) * d + b),
             as_u32(as_half2(__builtin_amdgcn_perm(HIGH, w1, 0x04010400u)) * d + b),
             as_u32(as_half2(__builtin_amdgcn_perm(HIGH, w1, 0x04030402u)) * d + b)}};
}

// Two tokens' codes of a V column (COLUMN dimensions each) as f16 pairs
// {token, next token}, one pair a dimension. c: the chunk's words (4 tokens).
template <int BITS, int COLUMN>
__device__ __forceinline__ void decode_v(const uint32_t *c, int pair, half2v d, half2v b, uint32_t (&out)[COLUMN]) {
    if constexpr (BITS == 4) {
        uint32_t low;
        if constexpr (COLUMN == 8) {
            const uint32_t a = c[2 * pair], e = c[2 * pair + 1];
            low = __builtin_amdgcn_perm(e, a, 0x05040100u);
            const uint32_t high = __builtin_amdgcn_perm(e, a, 0x07060302u);
            out[4] = as_u32(as_half2(nibbles<0>(high)) * d + b);
            out[5] = as_u32(as_half2(nibbles<1>(high)) * d + b);
            out[6] = as_u32(as_half2(nibbles<2>(high)) * d + b);
            out[7] = as_u32(as_half2(nibbles<3>(high)) * d + b);
        } else {
            low = c[pair];
        }
        out[0] = as_u32(as_half2(nibbles<0>(low)) * d + b);
        out[1] = as_u32(as_half2(nibbles<1>(low)) * d + b);
        out[2] = as_u32(as_half2(nibbles<2>(low)) * d + b);
        out[3] = as_u32(as_half2(nibbles<3>(low)) * d + b);
    } else {
        const uint32_t a = c[2 * pair], e = c[2 * pair + 1];
        out[0] = as_u32(as_half2(__builtin_amdgcn_perm(e, a, 0x0c040c00u) | 0x64006400u) * d + b);
        out[1] = as_u32(as_half2(__builtin_amdgcn_perm(e, a, 0x0c050c01u) | 0x64006400u) * d + b);
        out[2] = as_u32(as_half2(__builtin_amdgcn_perm(e, a, 0x0c060c02u) | 0x64006400u) * d + b);
        out[3] = as_u32(as_half2(__builtin_amdgcn_perm(e, a, 0x0c070c03u) | 0x64006400u) * d + b);
    }
}

__device__ __forceinline__ void store4(float *to, const float4 &x, float by) {
    *(float4 *)to = make_float4(x.x * by, x.y * by, x.z * by, x.w * by);
}
__device__ __forceinline__ void store4(_Float16 *to, const float4 &x, float by) {
    const half2v lo = {(_Float16)(x.x * by), (_Float16)(x.y * by)}, hi = {(_Float16)(x.z * by), (_Float16)(x.w * by)};
    *(uint2 *)to = make_uint2(as_u32(lo), as_u32(hi));
}

template <int BYTES> __device__ __forceinline__ void load_words(uint32_t *to, const uint8_t *p) {
    if constexpr (BYTES == 16) {
        const uint4 v = *(const uint4 *)p;
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    } else if constexpr (BYTES == 8) {
        const uint2 v = *(const uint2 *)p;
        to[0] = v.x, to[1] = v.y;
    } else {
        to[0] = *(const uint32_t *)p;
    }
}

// One tile (16 tokens of a KV head) as a lane holds it.
template <int BITS, int D> struct Tile {
    using G = CacheGeometry<BITS, D>;
    static constexpr int WORDS = G::CHUNK / 4;
    uint32_t k[G::UNITS][WORDS], v[G::UNITS][WORDS];
    uint32_t ks[G::GROUPS / 2];  // this lane's token's scales
    uint32_t vs[G::UNITS][2];    // its quad's scales in the group of its column

    __device__ __forceinline__ void load(const uint8_t *tile, int n, int h) {
#pragma unroll
        for (int u = 0; u < G::UNITS; ++u) {
            load_words<G::CHUNK>(k[u], tile + ((u * 16 + n) * 4 + h) * G::CHUNK);
            load_words<G::CHUNK>(v[u], tile + G::V_CODES + ((u * 4 + h) * 16 + n) * G::CHUNK);
            const int group = u * G::UNIT_GROUPS + n * G::COLUMN / 32;
            load_words<8>(vs[u], tile + G::V_SCALES + 8 * (h * G::GROUPS + group));
        }
        load_words<2 * G::GROUPS>(ks, tile + G::K_SCALES + 2 * n * G::GROUPS);
    }
    __device__ __forceinline__ half2v k_scale(int g) const {
        const half2v s = as_half2(ks[g >> 1]);
        return half2v{s[g & 1], s[g & 1]};
    }
    __device__ __forceinline__ Operand k_operand(int u, int gi, half2v d) const {
        const half2v b = bias_of<BITS>(d);
        if constexpr (BITS == 4) return decode_k4(k[u][gi], d, b);
        else return decode_k8(k[u][2 * gi], k[u][2 * gi + 1], d, b);
    }
    // Scales of the quad's tokens outside [from, to) become zero: never written
    // places may hold anything, a NaN scale among it.
    __device__ __forceinline__ void keep(int first, int from, int to) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            uint32_t mask = 0;
            if (first + 2 * p >= from && first + 2 * p < to) mask |= 0xffffu;
            if (first + 2 * p + 1 >= from && first + 2 * p + 1 < to) mask |= 0xffff0000u;
#pragma unroll
            for (int u = 0; u < G::UNITS; ++u) vs[u][p] &= mask;
        }
    }
};

// The tile index's place in the cache; `valid` is false for a page it lacks.
template <int BITS, int D>
__device__ __forceinline__ const uint8_t *tile_at(const CacheView &c, const int32_t *__restrict__ table, uint32_t head,
                                                  uint32_t tile, bool &valid) {
    const uint32_t page = (uint32_t)table[tile >> c.tiles_log2];
    valid = page < c.pages;
    const uint64_t at = (((uint64_t)(valid ? page : 0) * c.kv_heads + head) << c.tiles_log2) +
                        (tile & ((1u << c.tiles_log2) - 1u));
    return c.bytes + at * CacheGeometry<BITS, D>::TILE_BYTES;
}

// Over a row's four lanes (quarters h of lane / 16), by swaps of rows of lanes.
__device__ __forceinline__ float over_quarters_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float over_quarters_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What a workgroup works on.
struct Span {
    int rows;         // query rows of the (sequence, KV head)
    int first_row;    // of this workgroup
    int start;        // first query token of the sequence
    int position;     // of the sequence's first new token (negative: before its start)
    int from, to;     // tokens some row sees
    int low, high;    // steps of this split
};

// The query rows of sequence b, whatever `starts` holds.
__device__ __forceinline__ void rows_of(const AttentionArgs &a, uint32_t b, int &begin, int &tokens) {
    begin = (int)(b * a.max_tokens);
    tokens = (int)a.max_tokens;
    if (a.starts) {
        begin = min(max(a.starts[b], 0), (int)a.rows);
        tokens = min(min(max(a.starts[b + 1], begin), (int)a.rows) - begin, (int)a.max_tokens);
    }
}

// The rows and steps of a workgroup; false where it has no rows.
template <int ROWS, int STEP>
__device__ __forceinline__ bool span_of(const AttentionArgs &a, uint32_t b, uint32_t block, uint32_t split, Span &s) {
    int tokens;
    rows_of(a, b, s.start, tokens);
    s.rows = tokens * (int)a.group;
    s.first_row = (int)block * ROWS;
    if (s.first_row >= s.rows) return false;
    const int length = min(max(a.lengths[b], 0), (int)a.capacity);
    s.position = length - tokens;
    const int token_low = s.first_row / (int)a.group;
    const int token_high = min(s.first_row + ROWS - 1, s.rows - 1) / (int)a.group;
    s.to = max(s.position + token_high + 1, 0);
    // the window may be as large as an int holds: no sum may pass it
    s.from = a.window ? max(s.position + token_low - (int)a.window + 1, 0) : 0;
    const int begin_step = s.from / STEP, steps = s.to > s.from ? (s.to + STEP - 1) / STEP - begin_step : 0;
    const int each = (steps + (int)a.splits - 1) / (int)a.splits;
    s.low = begin_step + min((int)split * each, steps);
    s.high = begin_step + min(((int)split + 1) * each, steps);
    return true;
}

// RT tiles of 16 query rows in a wave: the lane of row n = lane % 16 and quarter
// h = lane / 16 holds Q^T as B operands (dimensions 32 g + 8 h ..+7 of a group), the
// row's statistics, and of O^T the dimensions u * UNIT_DIMS + (4 h + e) * COLUMN + j
// of unit u in o[..][u * COLUMN + j][e].
template <int BITS, int D, int RT, bool F32> struct Rows {
    using G = CacheGeometry<BITS, D>;
    using T = std::conditional_t<F32, float, _Float16>;
    static constexpr int GROUPS = G::GROUPS, PARTS = F32 ? 2 : 1, TILES_O = D / 16;
    Operand q[PARTS][RT][GROUPS];
    floatx4 o[RT][TILES_O];
    float scale[RT];               // of the scores (log2), the F32 row's own power of two among it
    float top[RT], sum[RT];        // reference maximum (log2), this lane's sum
    int position[RT], below[RT];   // a row sees below < j <= position
    int clear_from, clear_to;      // tokens [clear_from, clear_to) are seen by every live row
    int seen_from, seen_to;        // tokens some live row sees

    __device__ __forceinline__ void load(const AttentionArgs &a, const Span &s, uint32_t head, int first_row, int n,
                                         int h) {
        const int group = (int)a.group;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int row = first_row + 16 * t + n, token = row / group;
            const bool live = row < s.rows;
            const T *p = (const T *)a.q + (uint64_t)(s.start + token) * a.q_stride +
                         (head * a.group + row - token * group) * D;
            position[t] = live ? s.position + token : -1;
            below[t] = a.window ? s.position + token - (int)a.window : -1;
            scale[t] = a.scale;
            top[t] = LOWEST, sum[t] = 0.0f;
#pragma unroll
            for (int j = 0; j < TILES_O; ++j) o[t][j] = floatx4{0, 0, 0, 0};
            if constexpr (!F32) {
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (live) v = *(const uint4 *)(p + 32 * g + 8 * h);
                    q[0][t][g] = {{v.x, v.y, v.z, v.w}};
                }
            } else {
                float x[GROUPS][8];
                float most = 0.0f;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    float4 u = make_float4(0, 0, 0, 0), v = u;
                    if (live) u = ((const float4 *)(p + 32 * g + 8 * h))[0], v = ((const float4 *)(p + 32 * g + 8 * h))[1];
                    x[g][0] = u.x, x[g][1] = u.y, x[g][2] = u.z, x[g][3] = u.w;
                    x[g][4] = v.x, x[g][5] = v.y, x[g][6] = v.z, x[g][7] = v.w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[g][e]));
                }
                // the row's largest magnitude comes to [2^7, 2^8): hi + lo then hold 22 bits of it
                most = over_quarters_max(most);
                const uint32_t exponent = min(max(__float_as_uint(most) >> 23 & 255u, 8u), 254u);
                const float up = __uint_as_float((261u - exponent) << 23);
                // (never 0, which would turn a hidden score's -inf into NaN)
                scale[t] = fmaxf(scale[t] * __uint_as_float((exponent - 7u) << 23), 1.17549435e-38f);
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x0 = x[g][2 * e] * up, x1 = x[g][2 * e + 1] * up;
                        const half2v hi = {(_Float16)x0, (_Float16)x1};
                        const half2v lo = {(_Float16)(x0 - (float)hi[0]), (_Float16)(x1 - (float)hi[1])};
                        q[0][t][g].w[e] = as_u32(hi);
                        q[PARTS - 1][t][g].w[e] = as_u32(lo);
                    }
            }
        }
        const int low = s.position + first_row / group;
        const int high = s.position + (min(first_row + 16 * RT, s.rows) - 1) / group;
        clear_to = low + 1;
        clear_from = a.window ? max(high - (int)a.window + 1, 0) : 0;
        seen_to = first_row < s.rows ? high + 1 : 0;
        seen_from = a.window ? max(low - (int)a.window + 1, 0) : 0;
    }

    // S^T += K Q^T of one group
    __device__ __forceinline__ void score(half8 k, int g, floatx4 (&x)[RT]) const {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[p][t][g].get(), x[t], 0, 0, 0);
    }
    // O^T += V^T P^T of 16 dimensions
    __device__ __forceinline__ void add(half8 v, int j, const Operand (&p)[PARTS][RT]) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < PARTS; ++i)
                o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[i][t].get(), o[t][j], 0, 0, 0);
    }
    // Scores of the tokens first .. first + 3 (this lane's) that a row does not see become -inf.
    // (Bitwise on purpose: one select a score, no branches.)
    __device__ __forceinline__ void mask(floatx4 (&x)[RT], int first, bool valid) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int last = valid ? position[t] : -1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool hidden = (first + e > last) | (first + e <= below[t]);
                x[t][e] = hidden ? -__builtin_inff() : x[t][e];
            }
        }
    }
    // Weights of two tiles' raw scores, as the B operand of the next product.
    // The common step asks only whether any score passes its row's reference by
    // more than SLACK; the maximum over the row's lanes is taken where one does.
    __device__ __forceinline__ void weigh(const floatx4 (&a)[RT], const floatx4 (&b)[RT], Operand (&p)[PARTS][RT]) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float most = fmaxf(fmaxf(fmaxf(a[t][0], a[t][1]), fmaxf(a[t][2], a[t][3])),
                               fmaxf(fmaxf(b[t][0], b[t][1]), fmaxf(b[t][2], b[t][3]))) * scale[t];
            if (__any(most > top[t] + SLACK)) {
                most = over_quarters_max(most);
                const float higher = fmaxf(top[t], most), by = __builtin_amdgcn_exp2f(top[t] - higher);
                top[t] = higher;
                sum[t] *= by;
#pragma unroll
                for (int j = 0; j < TILES_O; ++j) o[t][j] *= by;
            }
            const float down = RAISE - top[t];
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(e < 4 ? a[t][e & 3] : b[t][e & 3], scale[t], down));
            sum[t] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const half2v hi = {(_Float16)w[2 * e], (_Float16)w[2 * e + 1]};
                p[0][t].w[e] = as_u32(hi);
                if constexpr (F32)
                    p[PARTS - 1][t].w[e] = as_u32(half2v{(_Float16)(w[2 * e] - (float)hi[0]),
                                                         (_Float16)(w[2 * e + 1] - (float)hi[1])});
            }
        }
    }
};

}  // namespace

}  // namespace nuq
