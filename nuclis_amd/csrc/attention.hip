// Attention of new queries over the quantised paged cache (layout: cache.h).
//
//   o[r] = sum_j softmax_j(scale * q[r] . K[j]) V[j],
//   j in (pos_r - window, pos_r] (all of [0, pos_r] without a window),
//   pos_r = length - new tokens + r
//
// Rows. The query rows of a KV head are its sequence's new tokens times the
// group of query heads that share it (row = token * group + head), so the
// cache is read once for a whole group. A wave holds RT tiles of 16 rows.
//
// Matrix form. S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: K and
// V are the A operands, decoded in registers straight from the lanes' wide
// loads; both results then have the row in lane % 16, so maxima, sums and
// rescaling never leave the lane but for two steps over its quarters, and P
// is V's B operand as it stands: its k order (token 4 h + e of the first tile,
// then of the second, h = lane / 16) is the order V's quads are loaded in.
//
// Precision. The cache's values are f16 numbers, so K and V enter exactly.
// F16 queries enter exactly too, and P is rounded to f16 once (a relative
// 2^-12 of each weight, as large as the rounding of the F16 output). F32
// queries are carried as two f16 parts after scaling each row by a power of two
// (22 bits at any magnitude), and P as two parts as well, so outputs keep F32
// precision. Scores, maxima, sums and outputs are F32. P is kept within
// [0, 2^15] relative to a reference that follows the row's maximum: it moves
// only when a score passes it by 2^8, so most steps rescale nothing.
//
// Rows without a token in reach (an empty sequence, positions before the
// sequence's start) are written as zeros. Positions on a page outside
// [0, pages) are not attended to.
//
// Work split. The four waves of a workgroup take steps of 32 tokens in turn and
// are merged in LDS; a long axis with few rows is split over workgroups, whose
// partial (maximum, sum, output) go to the workspace for a second kernel.
#include "attention.h"

#include <algorithm>

namespace nuq {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float LOWEST = -3.402823466e38f;  // a running maximum before any token
constexpr float RAISE = 7.0f;   // P is 2^RAISE at the reference
constexpr float SLACK = 8.0f;   // how far (log2) a score may pass the reference
constexpr int WAVES = 4, STEP = 32, MAX_SPLITS = 64;

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

__device__ __forceinline__ float over_quarters_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float over_quarters_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
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
template <int ROWS>
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

template <int BITS, int D, int RT, bool F32>
__global__ void __launch_bounds__(64 * WAVES, 2) attention_rows_kernel(CacheView c, AttentionArgs a) {
    using G = CacheGeometry<BITS, D>;
    using T = std::conditional_t<F32, float, _Float16>;
    constexpr int GROUPS = G::GROUPS, PARTS = F32 ? 2 : 1, TILES_O = D / 16;
    __shared__ __align__(16) float merge_o[WAVES][16][D + 4];
    __shared__ float merge_m[WAVES][16], merge_l[WAVES][16];

    const int lane = (int)threadIdx.x & 63, n = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // the KV head runs fastest: with 8 of them, the workgroups of one head (and
    // its share of the cache) stay on one XCD
    uint32_t id = blockIdx.x;
    const uint32_t head = id % c.kv_heads;
    id /= c.kv_heads;
    const uint32_t split = id % a.splits;
    id /= a.splits;
    const uint32_t block = a.blocks - 1 - id % a.blocks, b = id / a.blocks;  // long rows first
    Span s;
    if (!span_of<16 * RT>(a, b, block, split, s)) return;
    const int32_t *table = a.table + b * a.table_stride;

    // Q^T as B operands: lane (row n, quarter h) holds dimensions 32 g + 8 h ..+7
    Operand q[PARTS][RT][GROUPS];
    float scale[RT];
    int position[RT], below[RT];  // a row sees below < j <= position
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = s.first_row + 16 * t + n;
        const bool live = row < s.rows;
        const int token = row / (int)a.group;
        const T *p = (const T *)a.q + (uint64_t)(s.start + token) * a.q_stride +
                     (head * a.group + row - token * a.group) * D;
        position[t] = live ? s.position + token : -1;
        below[t] = a.window ? s.position + token - (int)a.window : -1;
        scale[t] = a.scale;
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
            scale[t] *= __uint_as_float((exponent - 7u) << 23);
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

    floatx4 o[RT][TILES_O];
    float top[RT], sum[RT];  // reference maximum (log2), this lane's sum
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        top[t] = LOWEST, sum[t] = 0.0f;
#pragma unroll
        for (int j = 0; j < TILES_O; ++j) o[t][j] = floatx4{0, 0, 0, 0};
    }
    // steps in [clear_from, clear_to) are seen by every row in full
    const int token_low = s.first_row / (int)a.group;
    const int token_high = min(s.first_row + 16 * RT - 1, s.rows - 1) / (int)a.group;
    const int clear_to = (s.position + token_low + 1) / STEP;  // may be 0 or negative
    const int clear_from = a.window ? (max(s.position + token_high - (int)a.window + 1, 0) + STEP - 1) / STEP : 0;

    Tile<BITS, D> next[2];
    bool next_valid[2];
    const auto fetch = [&](int step) {
        // the second half of the last step may lie past the table: it is masked, and reads the first half again
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tile = 2 * step + i;
            const bool inside = 16 * tile < s.to;
            next[i].load(tile_at<BITS, D>(c, table, head, (uint32_t)(inside ? tile : 2 * step), next_valid[i]), n, h);
        }
    };
    int step = s.low + wave;
    if (step < s.high) fetch(step);
    for (; step < s.high; step += WAVES) {
        Tile<BITS, D> tile[2] = {next[0], next[1]};
        const bool valid[2] = {next_valid[0], next_valid[1]};
        if (step + WAVES < s.high) fetch(step + WAVES);

        floatx4 x[RT][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int t = 0; t < RT; ++t) x[t][i] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const half8 k = tile[i].k_operand(g / G::UNIT_GROUPS, g % G::UNIT_GROUPS, tile[i].k_scale(g)).get();
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        x[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[p][t][g].get(), x[t][i], 0, 0, 0);
            }
        }
        const bool clear = step >= clear_from && step < clear_to && valid[0] && valid[1];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[t][i][e] *= scale[t];
        if (!clear) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int first = STEP * step + 16 * i + 4 * h;
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const int last = valid[i] ? position[t] : -1;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool hidden = (first + e > last) | (first + e <= below[t]);
                        x[t][i][e] = hidden ? -__builtin_inff() : x[t][i][e];
                    }
                }
                tile[i].keep(first, s.from, valid[i] ? s.to : 0);
            }
        }
        Operand p[PARTS][RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float most = fmaxf(fmaxf(fmaxf(x[t][0][0], x[t][0][1]), fmaxf(x[t][0][2], x[t][0][3])),
                               fmaxf(fmaxf(x[t][1][0], x[t][1][1]), fmaxf(x[t][1][2], x[t][1][3])));
            most = over_quarters_max(most);
            if (__any(most > top[t] + SLACK)) {
                const float higher = fmaxf(top[t], most);
                const float by = __builtin_amdgcn_exp2f(top[t] - higher);
                top[t] = higher;
                sum[t] *= by;
#pragma unroll
                for (int j = 0; j < TILES_O; ++j) o[t][j] *= by;
            }
            const float down = top[t] - RAISE;
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(x[t][e >> 2][e & 3] - down);
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
#pragma unroll
        for (int u = 0; u < G::UNITS; ++u) {
            uint32_t v[4][G::COLUMN];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const half2v d = as_half2(tile[k >> 1].vs[u][k & 1]);
                decode_v<BITS, G::COLUMN>(tile[k >> 1].v[u], k & 1, d, bias_of<BITS>(d), v[k]);
            }
#pragma unroll
            for (int j = 0; j < G::COLUMN; ++j) {
                const Operand av = {{v[0][j], v[1][j], v[2][j], v[3][j]}};
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int q_ = 0; q_ < PARTS; ++q_)
                        o[t][u * G::COLUMN + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            av.get(), p[q_][t].get(), o[t][u * G::COLUMN + j], 0, 0, 0);
            }
        }
    }

    // merge the waves: lane (row n, quarter h) holds, of unit u, the dimensions
    // u * UNIT_DIMS + (4 h + e) * COLUMN + j
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float l = over_quarters_sum(sum[t]);
        if (t) __syncthreads();
        if (h == 0) merge_m[wave][n] = top[t], merge_l[wave][n] = l;
#pragma unroll
        for (int u = 0; u < G::UNITS; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < G::COLUMN; j += 4) {
                    const int at = u * G::COLUMN + j;
                    *(float4 *)&merge_o[wave][n][u * G::UNIT_DIMS + (4 * h + e) * G::COLUMN + j] =
                        make_float4(o[t][at][e], o[t][at + 1][e], o[t][at + 2][e], o[t][at + 3][e]);
                }
        __syncthreads();
        // thread: row tid / 16, dimensions 4 * (tid % 16) + 64 i ..+3
        const int r = (int)threadIdx.x >> 4, row = s.first_row + 16 * t + r;
        if (row >= s.rows) continue;
        float m = merge_m[0][r];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = fmaxf(m, merge_m[w][r]);
        float by[WAVES], whole = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) by[w] = __builtin_amdgcn_exp2f(merge_m[w][r] - m), whole += by[w] * merge_l[w][r];
        const int token = row / (int)a.group;
        const uint64_t out_row = (uint64_t)(s.start + token);
        const uint32_t out_head = head * a.group + row - token * a.group;
        const float inverse = whole == 0.0f ? 0.0f : 1.0f / whole;
        float *partial = nullptr;
        if (a.splits > 1) {
            const uint64_t at = (out_row * (c.kv_heads * a.group) + out_head) * a.splits + split;
            partial = a.partial_o + at * D;
            if ((threadIdx.x & 15) == 0) a.partial_ml[2 * at] = m, a.partial_ml[2 * at + 1] = whole;
        }
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const int at = 4 * ((int)threadIdx.x & 15) + 64 * i;
            float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float4 y = *(const float4 *)&merge_o[w][r][at];
                x.x += by[w] * y.x, x.y += by[w] * y.y, x.z += by[w] * y.z, x.w += by[w] * y.w;
            }
            if (partial) {
                *(float4 *)(partial + at) = x;
            } else {
                store4((T *)a.out + out_row * a.out_stride + out_head * D + at, x, inverse);
            }
        }
    }
}

// Joins the splits of one (sequence, token, head) a workgroup: the first wave
// turns the splits' maxima into weights, then D / 4 threads take a split, 1024 / D
// splits at a time. A split without a token has sum 0 and no output: it is not
// read. (One wave walking 64 splits in order took 29 us after 32768 tokens,
// one round of memory latency a split; this takes 3.9.)
template <int D, bool F32>
__global__ void __launch_bounds__(256) attention_join_kernel(AttentionArgs a, uint32_t heads) {
    using T = std::conditional_t<F32, float, _Float16>;
    constexpr int ACROSS = D / 4, SIDE = 256 / ACROSS;
    __shared__ float weight[MAX_SPLITS], total;
    __shared__ __align__(16) float part[SIDE][D];
    const uint32_t head = blockIdx.x % heads, token = blockIdx.x / heads % a.max_tokens;
    const uint32_t b = blockIdx.x / heads / a.max_tokens;
    int begin, tokens;
    rows_of(a, b, begin, tokens);
    if ((int)token >= tokens) return;
    const uint64_t row = (uint64_t)begin + token, at = row * heads + head;
    const float *ml = a.partial_ml + 2 * at * a.splits;
    const uint32_t tid = threadIdx.x;
    if (tid < 64) {
        float m = LOWEST, l = 0.0f;
        if (tid < a.splits) m = ml[2 * tid], l = ml[2 * tid + 1];
        float top = m;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        const float w = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        float sum = l == 0.0f ? 0.0f : w * l;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        weight[tid] = l == 0.0f ? -1.0f : w;
        if (tid == 0) total = sum;
    }
    __syncthreads();
    const uint32_t side = tid / ACROSS, x4 = 4 * (tid % ACROSS);
    const float *p = a.partial_o + at * a.splits * D + x4;
    float4 x = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (uint32_t i = side; i < a.splits; i += SIDE) {
        const float w = weight[i];
        float4 y = make_float4(0, 0, 0, 0);
        if (w != -1.0f) y = *(const float4 *)(p + (uint64_t)i * D);
        x.x += w * y.x, x.y += w * y.y, x.z += w * y.z, x.w += w * y.w;
    }
    *(float4 *)&part[side][x4] = x;
    __syncthreads();
    if (tid >= ACROSS) return;
#pragma unroll
    for (int i = 1; i < SIDE; ++i) {
        const float4 y = *(const float4 *)&part[i][x4];
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    store4((T *)a.out + row * a.out_stride + head * D + x4, x, inverse);
}

template <int BITS, int D, int RT, bool F32>
hipError_t rows_launch(hipStream_t s, const CacheView &c, const AttentionArgs &a) {
    const uint32_t grid = c.kv_heads * a.splits * a.blocks * a.batch;
    attention_rows_kernel<BITS, D, RT, F32><<<grid, 64 * WAVES, 0, s>>>(c, a);
    return hipGetLastError();
}

template <int BITS, int D, bool F32> hipError_t rows_rt(hipStream_t s, const CacheView &c, const AttentionArgs &a) {
    if (a.row_tiles == 1) return rows_launch<BITS, D, 1, F32>(s, c, a);
    if constexpr (D <= 128 || !F32)
        if (a.row_tiles == 2) return rows_launch<BITS, D, 2, F32>(s, c, a);
    if constexpr (D <= 128 && !F32)
        if (a.row_tiles == 4) return rows_launch<BITS, D, 4, F32>(s, c, a);
    return hipErrorInvalidValue;
}

template <bool F32> hipError_t rows_dispatch(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t d,
                                             const AttentionArgs &a) {
#define NUQ_CASE(B, D) \
    if (bits == B && d == D) return rows_rt<B, D, F32>(s, c, a);
    NUQ_CASE(4, 64) NUQ_CASE(4, 128) NUQ_CASE(4, 256) NUQ_CASE(8, 64) NUQ_CASE(8, 128) NUQ_CASE(8, 256)
#undef NUQ_CASE
    return hipErrorInvalidValue;
}

}  // namespace

void plan_attention(uint32_t bits, uint32_t head_dim, uint32_t kv_heads, uint32_t f32, uint64_t max_length,
                    uint32_t heads, uint64_t max_floats, AttentionArgs *a) {
    (void)bits;
    const uint64_t rows = (uint64_t)a->max_tokens * a->group;
    uint32_t most = f32 ? (head_dim <= 128 ? 2 : 1) : (head_dim <= 128 ? 4 : 2);
    uint32_t tiles = 1;
    while (tiles < most && tiles * 16 < rows) tiles *= 2;
    a->row_tiles = tiles;
    a->blocks = (uint32_t)((rows + 16 * tiles - 1) / (16 * tiles));
    const uint64_t groups = (uint64_t)a->batch * kv_heads * a->blocks;
    uint64_t reach = max_length;
    if (a->window) reach = std::min<uint64_t>(reach, (uint64_t)a->window + a->max_tokens);
    // enough workgroups for two on every CU, each with at least one step a wave
    uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>((512 + groups - 1) / groups,
                                                              (reach + WAVES * STEP - 1) / (WAVES * STEP)));
    splits = std::min<uint64_t>(splits, MAX_SPLITS);
    const uint64_t each = (uint64_t)a->rows * heads * (head_dim + 2);
    if (splits > 1 && splits * each > max_floats) splits = std::max<uint64_t>(1, max_floats / each);
    a->splits = (uint32_t)splits;
    a->floats = splits > 1 ? splits * each : 0;
}

hipError_t launch_attention(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f32,
                            uint32_t heads, AttentionArgs a, float *work) {
    if (a.splits > 1) {
        a.partial_o = work;
        a.partial_ml = work + (uint64_t)a.rows * heads * a.splits * head_dim;
    }
    const hipError_t e = f32 ? rows_dispatch<true>(s, c, bits, head_dim, a) : rows_dispatch<false>(s, c, bits, head_dim, a);
    if (e != hipSuccess || a.splits == 1) return e;
    const uint32_t grid = a.batch * a.max_tokens * heads;
#define NUQ_CASE(D)                                                                                  \
    if (head_dim == D) {                                                                             \
        if (f32) attention_join_kernel<D, true><<<grid, 256, 0, s>>>(a, heads);                      \
        else attention_join_kernel<D, false><<<grid, 256, 0, s>>>(a, heads);                         \
    }
    NUQ_CASE(64) NUQ_CASE(128) NUQ_CASE(256)
#undef NUQ_CASE
    return hipGetLastError();
}

}  // namespace nuq
