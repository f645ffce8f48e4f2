// Attention of many new rows (prompts, chunks of them) over the quantised
// cache: the formulas, operands and precision of attention.hip, with the cache
// decoded once for the workgroup.
//
// Four waves hold 16 * RT query rows each. A step of TOKENS tokens is decoded to
// f16 operands in LDS by all four (each a quarter of K's and of V's operands,
// as one lane's wide load gives them), and read by all four: an operand is 64
// lanes of 16 bytes in lane order, so writes and reads are linear and free of
// bank conflicts. Two LDS buffers and one register stage: while a step is
// computed, the next is decoded from registers into the other buffer and the one
// after it is on its way from memory; one barrier a step.
//
// Why decoded through LDS: a step of 64 tokens costs about 400 vector
// instructions to decode, as many as the softmax of 64 rows; shared by four waves
// it is a quarter. RT is what two workgroups a CU leave room for in registers (O,
// Q and a step's scores), since one's products then run under the other's softmax.
// Operands are read from LDS ahead of their use.
//
// Measured (4096 tokens, 48 query heads of 128 over 8, F16, 4 bits): 239 us, 862
// TFLOP/s where a large f16 product reaches 1145 on the same card. The products alone
// take 153 us, the softmax adds 46 and the decode 53: what bounds it is the vector
// instructions between products (377 to 96 products a wave's step) that two waves
// a SIMD do not hide whole. Steps of 32 tokens, eight waves, two row tiles, and the
// next step's scores computed under this step's weights were each slower or equal.
#include "attention_tiles.h"

namespace nuq {

namespace {

template <int BITS, int D> struct Step {
    using G = CacheGeometry<BITS, D>;
    static constexpr int TOKENS = prompt_tokens(D);
    static constexpr int TILES = TOKENS / 16, PAIRS = TOKENS / 32;
    static constexpr int K_OPERANDS = TILES * G::GROUPS, V_OPERANDS = PAIRS * (D / 16);
    // a wave decodes K_ITEMS runs of K_SPAN groups of a token's chunk, and V_ITEMS dimensions of a V column
    static constexpr int K_SHARE = K_OPERANDS / WAVES, K_SPAN = K_SHARE < G::UNIT_GROUPS ? K_SHARE : G::UNIT_GROUPS;
    static constexpr int K_ITEMS = K_SHARE / K_SPAN, V_ITEMS = V_OPERANDS / WAVES;
    static constexpr int K_WORDS = K_SPAN * BITS / 4, V_WORDS = G::CHUNK / 4;
    static_assert(K_ITEMS * K_SPAN * WAVES == K_OPERANDS && V_ITEMS * WAVES == V_OPERANDS, "a wave's share is whole");
    static_assert(G::UNIT_GROUPS % K_SPAN == 0 && G::COLUMN % V_ITEMS == 0, "of one unit");
};

// A wave's share of a step between memory and LDS.
template <int BITS, int D> struct Raw {
    using S = Step<BITS, D>;
    using G = CacheGeometry<BITS, D>;
    uint32_t k[S::K_ITEMS][S::K_WORDS], ks[S::K_ITEMS][S::K_SPAN / 2];
    uint32_t v[2][S::V_WORDS], vs[2][2];
    uint32_t there;                     // bit i: the i-th K item's page exists; bits 30, 31: V's tiles' do
    uint32_t page[S::K_ITEMS + 2];      // of the next step to load, looked up a step before it

    // The step's tile `tile`; past the last token its first one, which is masked.
    static __device__ __forceinline__ uint32_t tile_of(int step, int tile, int to) {
        const int first = step * S::TILES;
        return (uint32_t)(first + (16 * (first + tile) < to ? tile : 0));
    }
    static __device__ __forceinline__ int k_tile(int wave, int i) {
        return (wave * S::K_SHARE + i * S::K_SPAN) / G::GROUPS;
    }
    static __device__ __forceinline__ int v_tile(int wave, int i) { return wave * S::V_ITEMS / (D / 16) * 2 + i; }

    __device__ __forceinline__ void look_up(const CacheView &c, PageTable table, int step, int to, int wave) {
#pragma unroll
        for (int i = 0; i < S::K_ITEMS + 2; ++i) {
            const int tile = i < S::K_ITEMS ? k_tile(wave, i) : v_tile(wave, i - S::K_ITEMS);
            page[i] = (uint32_t)table[tile_of(step, tile, to) >> c.tiles_log2];
        }
    }
    __device__ __forceinline__ void load(const CacheView &c, uint32_t head, int step, int to, int wave, int n, int h) {
        there = 0;
#pragma unroll
        for (int i = 0; i < S::K_ITEMS; ++i) {
            const int g = (wave * S::K_SHARE + i * S::K_SPAN) % G::GROUPS, u = g / G::UNIT_GROUPS;
            bool valid;
            const uint8_t *p = tile_at<BITS, D>(c, page[i], head, tile_of(step, k_tile(wave, i), to), valid);
            there |= (uint32_t)valid << i;
            load_words<S::K_SPAN * BITS>(k[i], p + u * 64 * G::CHUNK + g % G::UNIT_GROUPS * BITS,
                                         (uint32_t)(n * 4 + h) * G::CHUNK);
            load_words<2 * S::K_SPAN>(ks[i], p + G::K_SCALES + 2 * g, (uint32_t)(2 * n * G::GROUPS));
        }
        const int u = wave * S::V_ITEMS % (D / 16) / G::COLUMN;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bool valid;
            const uint8_t *p =
                tile_at<BITS, D>(c, page[S::K_ITEMS + i], head, tile_of(step, v_tile(wave, i), to), valid);
            there |= (uint32_t)valid << (30 + i);
            load_words<G::CHUNK>(v[i], p + G::V_CODES + u * 64 * G::CHUNK, (uint32_t)(h * 16 + n) * G::CHUNK);
            load_words<8>(vs[i], p + G::V_SCALES + 8 * u * G::UNIT_GROUPS,
                          (uint32_t)(8 * (h * G::GROUPS + n * G::COLUMN / 32)));
        }
    }

    // To LDS, V's scales of tokens outside [from, to) or on no page as zeros.
    __device__ __forceinline__ void decode(uint4 (*kb)[64], uint4 (*vb)[64], int step, int from, int to, int wave,
                                           int lane) const {
#pragma unroll
        for (int i = 0; i < S::K_ITEMS; ++i) {
#pragma unroll
            for (int g = 0; g < S::K_SPAN; ++g) {
                const half2v d = both(ks[i][g >> 1], g & 1), b = bias_of<BITS>(d);
                Operand o;
                if constexpr (BITS == 4) o = decode_k4(k[i][g], d, b);
                else o = decode_k8(k[i][2 * g], k[i][2 * g + 1], d, b);
                kb[wave * S::K_SHARE + i * S::K_SPAN + g][lane] = make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]);
            }
        }
        const int operand = wave * S::V_ITEMS, j0 = operand % G::COLUMN;
        const int first = S::TOKENS * step, v_first = first + 32 * (operand / (D / 16)) + 4 * (lane >> 4);
        const bool edge = first < from || first + S::TOKENS > to || there >> 30 != 3;
        uint32_t out[4][S::V_ITEMS];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int i = x >> 1, pair = x & 1;
            uint32_t scales = vs[i][pair];
            if (edge) {
                const int t = v_first + 16 * i + 2 * pair, end = (there >> (30 + i) & 1u) ? to : 0;
                uint32_t mask = 0;
                if (t >= from && t < end) mask |= 0xffffu;
                if (t + 1 >= from && t + 1 < end) mask |= 0xffff0000u;
                scales &= mask;
            }
            const half2v d = as_half2(scales), b = bias_of<BITS>(d);
            if constexpr (BITS == 4) {
                uint32_t w;  // four dimensions of two tokens, from j0 on
                if constexpr (G::COLUMN == 8)
                    w = __builtin_amdgcn_perm(v[i][2 * pair + 1], v[i][2 * pair], j0 & 4 ? 0x07060302u : 0x05040100u);
                else
                    w = v[i][pair];
                if constexpr (S::V_ITEMS == 2) w >>= 4 * (j0 & 3);
                out[x][0] = as_u32(as_half2(nibbles<0>(w)) * d + b);
                out[x][1] = as_u32(as_half2(nibbles<1>(w)) * d + b);
                if constexpr (S::V_ITEMS == 4) {
                    out[x][2] = as_u32(as_half2(nibbles<2>(w)) * d + b);
                    out[x][3] = as_u32(as_half2(nibbles<3>(w)) * d + b);
                }
            } else {
#pragma unroll
                for (int j = 0; j < S::V_ITEMS; ++j) {
                    const uint32_t pick = 0x0c040c00u + 0x00010001u * (uint32_t)(j0 + j);
                    const uint32_t w = __builtin_amdgcn_perm(v[i][2 * pair + 1], v[i][2 * pair], pick);
                    out[x][j] = as_u32(as_half2(w | 0x64006400u) * d + b);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < S::V_ITEMS; ++j)
            vb[operand + j][lane] = make_uint4(out[0][j], out[1][j], out[2][j], out[3][j]);
    }
};

template <int BITS, int D, int RT, bool F32>
__global__ void __launch_bounds__(64 * WAVES, 2) attention_prompt_kernel(CacheView c, AttentionArgs a) {
    using G = CacheGeometry<BITS, D>;
    using S = Step<BITS, D>;
    using T = std::conditional_t<F32, float, _Float16>;
    constexpr int PARTS = F32 ? 2 : 1;
    // LDS operands on their way; one where O and Q leave no registers for two (8 bits: 251 us for a
    // prompt of 4096 with 16 heads of 256, 460 with two of them spilling; at 4 bits two
    // are as fast, 149 and 151 us for two chunks of 1000 over a window)
    constexpr int AHEAD = D == 256 && BITS == 8 && !F32 ? 1 : 2;
    __shared__ uint4 kb[2][S::K_OPERANDS][64], vb[2][S::V_OPERANDS][64];
    __shared__ int valid[2][4];  // of a buffer's tiles

    const int lane = (int)threadIdx.x & 63, n = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    uint32_t id = blockIdx.x;  // as in attention_rows_kernel
    const uint32_t head = id % c.kv_heads;
    id /= c.kv_heads;
    const uint32_t split = id % a.splits;
    id /= a.splits;
    uint32_t b = id / a.blocks, place = id % a.blocks, blocks = a.blocks;
    if (a.starts) {
        place = id;
        if (!place_of(a, a.group, 16 * RT * WAVES, place, b, blocks)) return;
    }
    const uint32_t block = blocks - 1 - place;
    Span s;
    if (!span_of<16 * RT * WAVES, S::TOKENS>(a, b, block, split, s)) return;
    const PageTable table = table_of(a, b);

    const int first_row = s.first_row + 16 * RT * wave;
    Rows<BITS, D, RT, F32> rows;
    typename Rows<BITS, D, RT, F32>::Raw queries;
    rows.load(a, s, head, first_row, n, h, queries);

    Raw<BITS, D> raw;
    const auto decode = [&](int step, int buffer) {
#pragma unroll
        for (int i = 0; i < S::K_ITEMS; ++i)
            if (lane == 0) valid[buffer][raw.k_tile(wave, i)] = (int)(raw.there >> i & 1u);
        raw.decode(kb[buffer], vb[buffer], step, s.from, s.to, wave, lane);
    };
    const int last = max(s.high - 1, 0);
    raw.look_up(c, table, min(s.low, last), s.to, wave);
    raw.load(c, head, min(s.low, last), s.to, wave, n, h);
    raw.look_up(c, table, min(s.low + 1, last), s.to, wave);
    rows.prepare(queries);
    if (s.low < s.high) {
        decode(s.low, 0);
        raw.load(c, head, min(s.low + 1, last), s.to, wave, n, h);
        raw.look_up(c, table, min(s.low + 2, last), s.to, wave);
        __syncthreads();
    }
    for (int step = s.low; step < s.high; ++step) {
        const int buffer = (step - s.low) & 1, first = S::TOKENS * step;
        int there[S::TILES];
        bool all = true;
#pragma unroll
        for (int i = 0; i < S::TILES; ++i) there[i] = valid[buffer][i];
        if (step + 1 < s.high) {
            decode(step + 1, buffer ^ 1);
            raw.load(c, head, min(step + 2, last), s.to, wave, n, h);
            raw.look_up(c, table, min(step + 3, last), s.to, wave);
        }
        if (first < rows.seen_to && first + S::TOKENS > rows.seen_from) {
#pragma unroll
            for (int i = 0; i < S::TILES; ++i) {
                there[i] = __builtin_amdgcn_readfirstlane(there[i]);
                all &= there[i] != 0;
            }
            const bool masked = first < rows.clear_from || first + S::TOKENS > rows.clear_to || !all;
#pragma unroll
            for (int pair = 0; pair < S::PAIRS; ++pair) {
                floatx4 x[2][RT];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int t = 0; t < RT; ++t) x[i][t] = floatx4{0, 0, 0, 0};
                const uint4(*const k)[64] = kb[buffer] + 2 * pair * G::GROUPS;
                const uint4(*const v)[64] = vb[buffer] + pair * (D / 16);
                __builtin_amdgcn_sched_barrier(0);
                uint4 ahead[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) ahead[i] = k[i][lane];
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
                for (int i = 0; i < 2 * G::GROUPS; ++i) {
                    const uint4 now = ahead[i % AHEAD];
                    if (i + AHEAD < 2 * G::GROUPS) ahead[i % AHEAD] = k[i + AHEAD][lane];
                    rows.score(__builtin_bit_cast(half8, now), i % G::GROUPS, x[i / G::GROUPS]);
                    __builtin_amdgcn_sched_group_barrier(0x008, RT * PARTS, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        rows.mask(x[i], first + 32 * pair + 16 * i + 4 * h, there[2 * pair + i]);
                }
                Operand p[PARTS][RT];
                rows.template raise<2>(x);
                rows.template weigh<2>(x, p);
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) ahead[j] = v[j][lane];
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 1);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const uint4 now = ahead[j % AHEAD];
                    if (j + AHEAD < D / 16) ahead[j % AHEAD] = v[j + AHEAD][lane];
                    rows.template add<2>(__builtin_bit_cast(Operand, now), j, p);
                    __builtin_amdgcn_sched_group_barrier(0x008, RT * PARTS, 1);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
                }
            }
        }
        __syncthreads();
    }

#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float l = over_quarters_sum(rows.sum[t]);
        const int row = first_row + 16 * t + n;
        if (row >= s.rows) continue;
        const int token = row / (int)a.group;
        const uint64_t out_row = (uint64_t)(s.start + token);
        const uint32_t out_head = head * a.group + row - token * a.group;
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        const uint64_t at =
            (partial_row(a, b, s.start, token) * (c.kv_heads * a.group) + out_head) * a.splits + split;
        if (a.splits > 1 && h == 0) a.partial_ml[2 * at] = rows.top[t], a.partial_ml[2 * at + 1] = l;
#pragma unroll
        for (int u = 0; u < G::UNITS; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < G::COLUMN; j += 4) {
                    const int o = u * G::COLUMN + j, dim = u * G::UNIT_DIMS + (4 * h + e) * G::COLUMN + j;
                    const float4 x = make_float4(rows.o[t][o][e], rows.o[t][o + 1][e], rows.o[t][o + 2][e],
                                                 rows.o[t][o + 3][e]);
                    if (a.splits > 1) *(float4 *)(a.partial_o + at * D + dim) = x;
                    else store4((T *)a.out + out_row * a.out_stride + out_head * D + dim, x, inverse);
                }
    }
}

template <int BITS, int D, bool F32> hipError_t prompt_launch(hipStream_t s, const CacheView &c, const AttentionArgs &a) {
    constexpr int RT = prompt_row_tiles(D, F32);
    const uint32_t grid = (uint32_t)(c.kv_heads * a.splits * a.units);
    attention_prompt_kernel<BITS, D, RT, F32><<<grid, 64 * WAVES, 0, s>>>(c, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_prompt(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t d, uint32_t f32,
                                   const AttentionArgs &a) {
#define NUQ_CASE(B, D) \
    if (bits == B && d == D) return f32 ? prompt_launch<B, D, true>(s, c, a) : prompt_launch<B, D, false>(s, c, a);
    NUQ_CASE(4, 64) NUQ_CASE(4, 128) NUQ_CASE(4, 256) NUQ_CASE(8, 64) NUQ_CASE(8, 128) NUQ_CASE(8, 256)
#undef NUQ_CASE
    return hipErrorInvalidValue;
}

}  // namespace nuq
