// What the attention kernels share: the cache's tiles as matrix operands, and the
// rows and steps a workgroup works on (attention.hip, attention_prompt.hip).
#pragma once

#include "attention.h"

namespace nuq {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float LOWEST = -3.402823466e38f;  // a running maximum before any token
constexpr float RAISE = 7.0f;   // P is 2^RAISE at the reference
constexpr float SLACK = 8.0f;   // how far (log2) a score may pass the reference
constexpr int WAVES = 4, MAX_SPLITS = 64;

__device__ __forceinline__ half2v as_half2(uint32_t u) { return __builtin_bit_cast(half2v, u); }
__device__ __forceinline__ uint32_t as_u32(half2v h) { return __builtin_bit_cast(uint32_t, h); }

// What rounding x0, x1 to `hi` left over: x - (float)hi in one instruction each.
__device__ __forceinline__ half2v rest_of(half2v hi, float x0, float x1) {
    float a, b;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(as_u32(hi)), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(as_u32(hi)), "v"(x1));
    return half2v{(_Float16)a, (_Float16)b};
}

struct Operand {  // 8 f16 of one lane
    uint32_t w[4];
    __device__ __forceinline__ half8 get() const { return __builtin_bit_cast(half8, *this); }
    __device__ __forceinline__ half4 low() const { return __builtin_shufflevector(get(), get(), 0, 1, 2, 3); }
};

// A pair of one of a pair's halves. (No subscript that a loop makes: it kept whole
// structs in memory.)
__device__ __forceinline__ half2v both(uint32_t pair, int which) {
    const half2v s = as_half2(pair);
    return which ? half2v{s[1], s[1]} : half2v{s[0], s[0]};
}

// (x & mask) | bits as the one instruction it is: it takes one constant from a
// scalar register, so the compiler, left to itself, keeps both there and issues two.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t out;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(out) : "v"(x), "s"(mask), "v"(bits));
    return out;
}

// A nibble in the top mantissa bits of 16.0 is 16 + code; a byte under 0x64 is
// 1024 + code. One f16 fma by (d, -bias d) then gives d * (code - offset) exactly.
template <int BITS> __device__ __forceinline__ half2v bias_of(half2v d) {
    return d * (_Float16)(BITS == 4 ? -24.0f : -1152.0f);
}
// The pair of nibbles at bits p and 16 + p, p = 4 I.
template <int I> __device__ __forceinline__ uint32_t nibbles(uint32_t w) {
    constexpr int SHIFT = 6 - 4 * I;
    const uint32_t s = SHIFT >= 0 ? w << (SHIFT >= 0 ? SHIFT : 0) : w >> (SHIFT >= 0 ? 0 : -SHIFT);
    return and_or(s, 0x03c003c0u, 0x4c004c00u);
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

template <int BYTES> __device__ __forceinline__ void load_words(uint32_t *to, const uint8_t *base, uint32_t offset) {
    // (kept from being widened outside a loop: the load then takes the base from
    // scalar registers and adds these 32 bits itself)
    asm volatile("" : "+v"(offset));
    const uint8_t *p = base + offset;
    static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16);
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
            load_words<G::CHUNK>(k[u], tile + u * 64 * G::CHUNK, (uint32_t)(n * 4 + h) * G::CHUNK);
            load_words<G::CHUNK>(v[u], tile + G::V_CODES + u * 64 * G::CHUNK, (uint32_t)(h * 16 + n) * G::CHUNK);
            load_words<8>(vs[u], tile + G::V_SCALES + 8 * u * G::UNIT_GROUPS,
                          (uint32_t)(8 * (h * G::GROUPS + n * G::COLUMN / 32)));
        }
        load_words<2 * G::GROUPS>(ks, tile + G::K_SCALES, (uint32_t)(2 * n * G::GROUPS));
    }
    __device__ __forceinline__ half2v k_scale(int g) const { return both(ks[g >> 1], g & 1); }
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

// A sequence's row of the page table, which nothing writes meanwhile: read by scalar loads.
typedef const __attribute__((address_space(4))) int32_t *PageTable;
__device__ __forceinline__ PageTable table_of(const AttentionArgs &a, uint32_t b) {
    return (PageTable)(uintptr_t)(a.table + b * a.table_stride);
}

// The place of tile `tile` of its sequence, on page `page`; `valid` is false for a page the cache lacks.
template <int BITS, int D>
__device__ __forceinline__ const uint8_t *tile_at(const CacheView &c, uint32_t page, uint32_t head, uint32_t tile,
                                                  bool &valid) {
    valid = page < c.pages;
    const uint64_t at = (((uint64_t)(valid ? page : 0) * c.kv_heads + head) << c.tiles_log2) +
                        (tile & ((1u << c.tiles_log2) - 1u));
    // one for the wave, in scalar registers: loads take a 32-bit offset a lane beside it
    const uint64_t from = at * CacheGeometry<BITS, D>::TILE_BYTES;
    return c.bytes + ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(from >> 32)) << 32 |
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)from));
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

// The query rows of sequence b, whatever `starts` holds. `brought` are its new tokens, of
// which the first `tokens` have rows that are computed: they stand before the others.
__device__ __forceinline__ void rows_of(const AttentionArgs &a, uint32_t b, int &begin, int &tokens, int &brought) {
    begin = (int)(b * a.max_tokens);
    tokens = brought = (int)a.max_tokens;
    if (a.starts) {
        begin = min(max(a.starts[b], 0), (int)a.rows);
        const int end = max(a.starts[b + 1], begin);
        brought = end - begin;
        tokens = min(min(end, (int)a.rows) - begin, (int)a.max_tokens);
        if (tokens <= (int)a.above || tokens > (int)a.upto) tokens = 0;
    }
}

// Where the partial results of a (sequence, token) lie: by its query row, or where the plan
// is of few tokens a sequence by its place among those.
__device__ __forceinline__ uint64_t partial_row(const AttentionArgs &a, uint32_t b, int begin, int token) {
    return a.upto < a.max_tokens ? (uint64_t)b * a.upto + token : (uint64_t)(begin + token);
}

// The sequence and the place in it of unit `at`, where sequences of different counts of
// tokens have ceil(tokens * by / of) units each, one's behind the other's: `at` and
// `count` become the place and the sequence's units. False past the last. A lane
// counts a sequence's; without this a batch's short sequences leave most of a grid idle
// (a prompt of 1000 among 63 single tokens: 49 thousand workgroups, 29 us to pass over).
__device__ __forceinline__ bool place_of(const AttentionArgs &a, uint32_t by, uint32_t of, uint32_t &at, uint32_t &b,
                                         uint32_t &count) {
    const int lane = (int)threadIdx.x & 63;
    for (uint32_t first = 0; first < a.batch; first += 64) {
        int begin, tokens = 0, brought;
        if (first + lane < a.batch) rows_of(a, first + lane, begin, tokens, brought);
        const uint32_t own = ((uint32_t)tokens * by + of - 1) / of;
        uint32_t sum = own;  // of this lane's and all before it
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const uint32_t before = (uint32_t)__shfl_up((int)sum, off, 64);
            sum += lane >= off ? before : 0;
        }
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        if (at < all) {
            const int l = __builtin_ctzll(__ballot(sum > at));
            count = (uint32_t)__builtin_amdgcn_readlane((int)own, l);
            at -= (uint32_t)__builtin_amdgcn_readlane((int)sum, l) - count;
            b = first + l;
            return true;
        }
        at -= all;
    }
    return false;
}

// The rows and steps of a workgroup; false where it has no rows.
template <int ROWS, int STEP>
__device__ __forceinline__ bool span_of(const AttentionArgs &a, uint32_t b, uint32_t block, uint32_t split, Span &s) {
    int tokens, brought;
    rows_of(a, b, s.start, tokens, brought);
    s.rows = tokens * (int)a.group;
    s.first_row = (int)block * ROWS;
    if (s.first_row >= s.rows) return false;
    const int length = min(max(a.lengths[b], 0), (int)a.capacity);
    // (a start before -tokens leaves the rows nothing, as -tokens does)
    s.position = length - min(brought, length + tokens);
    const int token_low = s.first_row / (int)a.group;
    const int token_high = min(s.first_row + ROWS - 1, s.rows - 1) / (int)a.group;
    s.to = max(s.position + token_high + 1, 0);
    // the window may be as large as an int holds: no sum may pass it
    s.from = a.window ? max(s.position + token_low - (int)a.window + 1, 0) : 0;
    const int begin_step = s.to > s.from ? s.from / STEP : 0;
    const int steps = s.to > s.from ? (s.to + STEP - 1) / STEP - begin_step : 0;
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

    // Query rows as they are in memory, before `prepare` makes them operands (F32)
    // (F16: they are operands as they come).
    struct Raw {
        float4 x[F32 ? RT : 1][F32 ? GROUPS : 1][2];
    };

    // Requests the rows and sets their positions.
    __device__ __forceinline__ void load(const AttentionArgs &a, const Span &s, uint32_t head, int first_row, int n,
                                         int h, Raw &raw) {
        const int group = (int)a.group;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            // (rows past the last are its copies: their results are not written, and loads
            // without a branch around them leave the compiler exact counts to wait for)
            const int row = min(first_row + 16 * t + n, s.rows - 1), token = row / group;
            const T *p = (const T *)a.q + (uint64_t)(s.start + token) * a.q_stride +
                         (head * a.group + row - token * group) * D;
            position[t] = s.position + token;
            below[t] = a.window ? s.position + token - (int)a.window : -1;
            scale[t] = a.scale;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                if constexpr (F32) {
                    raw.x[t][g][0] = ((const float4 *)(p + 32 * g + 8 * h))[0];
                    raw.x[t][g][1] = ((const float4 *)(p + 32 * g + 8 * h))[1];
                } else {
                    const uint4 v = *(const uint4 *)(p + 32 * g + 8 * h);
                    q[0][t][g] = {{v.x, v.y, v.z, v.w}};
                }
            }
        }
        const int low = s.position + min(first_row, s.rows - 1) / group;
        const int high = s.position + (min(first_row + 16 * RT, s.rows) - 1) / group;
        clear_to = low + 1;
        clear_from = a.window ? max(high - (int)a.window + 1, 0) : 0;
        seen_to = first_row < s.rows ? high + 1 : 0;
        seen_from = a.window ? max(low - (int)a.window + 1, 0) : 0;
    }

    __device__ __forceinline__ void prepare(const Raw &raw) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            top[t] = LOWEST, sum[t] = 0.0f;
#pragma unroll
            for (int j = 0; j < TILES_O; ++j) o[t][j] = floatx4{0, 0, 0, 0};
            if constexpr (!F32) {
                // waited for here: left to their first use, in the loop, they would be waited for
                // in every turn of it, and with them the loads on their way
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // infinities become NaN, as the parts of an F32 query do: scores of -inf would
                        // make the row one that sees nothing
                        const half2v x = as_half2(q[0][t][g].w[e]);
                        q[0][t][g].w[e] = as_u32(x * (_Float16)0.0f + x);
                        asm volatile("" : "+v"(q[0][t][g].w[e]));
                    }
            } else {
                float most = 0.0f;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float4 &x = raw.x[t][g][i];
                        most = fmaxf(fmaxf(fmaxf(most, fabsf(x.x)), fmaxf(fabsf(x.y), fabsf(x.z))), fabsf(x.w));
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
                        const float4 &x = raw.x[t][g][e >> 1];
                        const float x0 = ((e & 1) ? x.z : x.x) * up, x1 = ((e & 1) ? x.w : x.y) * up;
                        const half2v hi = {(_Float16)x0, (_Float16)x1};
                        const half2v lo = rest_of(hi, x0, x1);
                        q[0][t][g].w[e] = as_u32(hi);
                        q[PARTS - 1][t][g].w[e] = as_u32(lo);
                    }
            }
        }
    }

    // S^T += K Q^T of one group
    __device__ __forceinline__ void score(half8 k, int g, floatx4 (&x)[RT]) const {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[p][t][g].get(), x[t], 0, 0, 0);
    }
    // O^T += V^T P^T of 16 dimensions, over two tiles' tokens (k = 32) or one's (k = 16)
    template <int TILES> __device__ __forceinline__ void add(const Operand &v, int j, const Operand (&p)[PARTS][RT]) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                if constexpr (TILES == 2)
                    o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.get(), p[i][t].get(), o[t][j], 0, 0, 0);
                else
                    o[t][j] = __builtin_amdgcn_mfma_f32_16x16x16f16(v.low(), p[i][t].low(), o[t][j], 0, 0, 0);
            }
    }
    // Scores of the tokens first .. first + 3 (this lane's) that a row does not see become -inf.
    // (Bitwise on purpose: one select a score, no branches. Written as `if (!valid || ... || ...) x = -inf`, a
    // uniform condition before two of the lanes', the compiler leaves the last score's move of a tile in the
    // uniform condition's block alone; the lanes' own block is empty, and they keep what they should not see.)
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
    // Moves the references of rows that a step's raw scores pass by more than SLACK.
    // The common step asks only whether one does; the maximum over a row's lanes
    // is taken where so.
    template <int TILES> __device__ __forceinline__ void raise(const floatx4 (&x)[TILES][RT]) {
        float most[RT];
        bool past = false;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            most[t] = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < TILES; ++i)
                most[t] = fmaxf(most[t], fmaxf(fmaxf(x[i][t][0], x[i][t][1]), fmaxf(x[i][t][2], x[i][t][3])));
            most[t] *= scale[t];
            past |= most[t] > top[t] + SLACK;
        }
        if (__any(past)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const float higher = fmaxf(top[t], over_quarters_max(most[t]));
                const float by = __builtin_amdgcn_exp2f(top[t] - higher);
                top[t] = higher;
                sum[t] *= by;
#pragma unroll
                for (int j = 0; j < TILES_O; ++j) o[t][j] *= by;
            }
        }
    }
    // Weights of one or two tiles' raw scores as the B operand of the next product.
    template <int TILES> __device__ __forceinline__ void weigh(const floatx4 (&x)[TILES][RT], Operand (&p)[PARTS][RT]) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float down = RAISE - top[t];
            float w[4 * TILES];
#pragma unroll
            for (int e = 0; e < 4 * TILES; ++e)
                w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e >> 2][t][e & 3], scale[t], down));
#pragma unroll
            for (int i = 0; i < TILES; ++i) sum[t] += (w[4 * i] + w[4 * i + 1]) + (w[4 * i + 2] + w[4 * i + 3]);
#pragma unroll
            for (int e = 0; e < 2 * TILES; ++e) {
                const half2v hi = {(_Float16)w[2 * e], (_Float16)w[2 * e + 1]};
                p[0][t].w[e] = as_u32(hi);
                if constexpr (F32) p[PARTS - 1][t].w[e] = as_u32(rest_of(hi, w[2 * e], w[2 * e + 1]));
            }
        }
    }
};

}  // namespace

}  // namespace nuq
