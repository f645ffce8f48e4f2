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
// 2^-11 of each weight, as large as the rounding of the F16 output). F32
// queries are carried as two f16 parts after scaling each row by a power of two
// (22 bits at any magnitude), and P as two parts as well: 22 bits of each weight, or
// 2^-32 of the row's sum where that is more, f16's smallest step against the
// 2^RAISE of the row's largest weight. Scores, maxima, sums and outputs are F32. P is kept within
// [0, 2^15] relative to a reference that follows the row's maximum: it moves
// only when a score passes it by 2^8, so most steps rescale nothing.
//
// Rows without a token in reach (an empty sequence, positions before the
// sequence's start) are written as zeros. Positions on a page outside
// [0, pages) are not attended to.
//
// Work split. The four waves of a workgroup take steps of 32 tokens (16 where two
// steps of 32 do not fit the registers, step_tiles) in turn and are merged in LDS; a
// long axis with few rows is split over workgroups, whose partial (maximum, sum,
// output) go to the workspace for a second kernel.
//
// Measured (48 query heads of 128 over 8, 4 bits), kernel by kernel in a trace. One F32
// token after 300 tokens: 7.0 us, a chain of four trips to memory; after 32768: 14.1 us and 3.9
// for the second kernel (37.8 MB, which a plain stream of that size reads in 7.1 us; a call among
// others takes 15.4, so part of a traced kernel's start and end is hidden there). 32 sequences of
// one F16 token up to 16384: 69 and 4.7 us, 4.6 TB/s in all, with the vector units half busy
// (F32 78 us a call). 4 x 8 F32 tokens up to 8191 at 8 bits: 24.3 and 4.0 us (25.4 a call, F16 20.9),
// latency and the decode of two blocks of rows.
#include "attention_tiles.h"

#include <algorithm>

namespace nuq {

namespace {

// Registers of a wave beside its steps in work and on their way: O, Q, and a step's scores, weights and decoded V.
constexpr int held_registers(int bits, int d, int rt, bool f32, int tiles) {
    const int parts = f32 ? 2 : 1, column = bits == 4 && d > 64 ? 8 : 4;
    return rt * d / 4 + rt * parts * d / 8 + tiles * (4 * rt + 2 * rt * parts + 2 * column) + 30;
}
// A tile's registers (struct Tile).
constexpr int tile_registers(int bits, int d) {
    const int units = d * bits / 32 <= 16 ? 1 : d * bits / 512;
    return 2 * (d * bits / 128) + d / 64 + 2 * units;
}
// A wave's step is two tiles of 16 tokens, or one where two such steps on their
// way do not fit 256 registers (two waves a SIMD).
constexpr int step_tiles(int bits, int d, int rt, bool f32) {
    return held_registers(bits, d, rt, f32, 2) + 4 * tile_registers(bits, d) <= 240 ? 2 : 1;
}
template <int BITS, int D, int RT, bool F32>
__global__ void __launch_bounds__(64 * WAVES, 2) attention_rows_kernel(CacheView c, AttentionArgs a) {
    using G = CacheGeometry<BITS, D>;
    using T = std::conditional_t<F32, float, _Float16>;
    constexpr int PARTS = F32 ? 2 : 1;
    constexpr int TILES = step_tiles(BITS, D, RT, F32), STEP = 16 * TILES;
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
    if (!span_of<16 * RT, STEP>(a, b, block, split, s)) return;
    const PageTable table = table_of(a, b);

    Rows<BITS, D, RT, F32> rows;
    typename Rows<BITS, D, RT, F32>::Raw queries;
    rows.load(a, s, head, s.first_row, n, h, queries);

    // Two steps ahead a wave looks up the pages, one step ahead it requests the tiles. The
    // second half of the last step may lie past the table: it is masked, and reads the first half again.
    Tile<BITS, D> next[TILES];
    bool next_valid[TILES];
    uint32_t page[TILES];
    const auto tile_of = [&](int step, int i) {
        const int first = TILES * step;
        return (uint32_t)(16 * (first + i) < s.to ? first + i : first);
    };
    const auto look_up = [&](int step) {
#pragma unroll
        for (int i = 0; i < TILES; ++i) page[i] = (uint32_t)table[tile_of(step, i) >> c.tiles_log2];
    };
    const auto fetch = [&](int step) {
#pragma unroll
        for (int i = 0; i < TILES; ++i)
            next[i].load(tile_at<BITS, D>(c, page[i], head, tile_of(step, i), next_valid[i]), n, h);
    };
    const int first_step = s.low + wave;
    // (the queries' F32 values and a step under way do not fit where rows are many or wide)
    if constexpr (F32 && RT * D > 128) rows.prepare(queries);
    // Loads stand under no condition, so that the compiler knows what to wait for:
    // past its last step a wave asks for that one again.
    const int last = max(s.high - 1, 0);
    look_up(min(first_step, last));
    fetch(min(first_step, last));
    look_up(min(first_step + WAVES, last));
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!F32 || RT * D <= 128) rows.prepare(queries);
    for (int step = first_step; step < s.high; step += WAVES) {
        Tile<BITS, D> tile[TILES];
        bool valid[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) tile[i] = next[i], valid[i] = next_valid[i];
        fetch(min(step + WAVES, last));
        look_up(min(step + 2 * WAVES, last));
        floatx4 x[TILES][RT];
        bool whole = true;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            whole &= valid[i];
#pragma unroll
            for (int t = 0; t < RT; ++t) x[i][t] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < G::GROUPS; ++g)
                rows.score(tile[i].k_operand(g / G::UNIT_GROUPS, g % G::UNIT_GROUPS, tile[i].k_scale(g)).get(), g,
                           x[i]);
        }
        if (STEP * step < rows.clear_from || STEP * (step + 1) > rows.clear_to || !whole) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const int first = STEP * step + 16 * i + 4 * h;
                rows.mask(x[i], first, valid[i]);
                tile[i].keep(first, s.from, valid[i] ? s.to : 0);
            }
        }
        Operand p[PARTS][RT];
        rows.template raise<TILES>(x);
        rows.template weigh<TILES>(x, p);
#pragma unroll
        for (int u = 0; u < G::UNITS; ++u) {
            uint32_t v[2 * TILES][G::COLUMN];
#pragma unroll
            for (int i = 0; i < 2 * TILES; ++i) {
                const half2v d = as_half2(tile[i >> 1].vs[u][i & 1]);
                decode_v<BITS, G::COLUMN>(tile[i >> 1].v[u], i & 1, d, bias_of<BITS>(d), v[i]);
            }
#pragma unroll
            for (int j = 0; j < G::COLUMN; ++j) {
                Operand av;
#pragma unroll
                for (int i = 0; i < 2 * TILES; ++i) av.w[i] = v[i][j];
                rows.template add<TILES>(av, u * G::COLUMN + j, p);
            }
        }
    }

    // merge the waves
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float l = over_quarters_sum(rows.sum[t]);
        if (t) __syncthreads();
        if (h == 0) merge_m[wave][n] = rows.top[t], merge_l[wave][n] = l;
#pragma unroll
        for (int u = 0; u < G::UNITS; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < G::COLUMN; j += 4) {
                    const int at = u * G::COLUMN + j;
                    *(float4 *)&merge_o[wave][n][u * G::UNIT_DIMS + (4 * h + e) * G::COLUMN + j] =
                        make_float4(rows.o[t][at][e], rows.o[t][at + 1][e], rows.o[t][at + 2][e],
                                    rows.o[t][at + 3][e]);
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
        for (int w = 0; w < WAVES; ++w) {
            by[w] = __builtin_amdgcn_exp2f(merge_m[w][r] - m);
            whole += by[w] * merge_l[w][r];
        }
        const int token = row / (int)a.group;
        const uint64_t out_row = (uint64_t)(s.start + token);
        const uint32_t out_head = head * a.group + row - token * a.group;
        const float inverse = whole == 0.0f ? 0.0f : 1.0f / whole;
        float *partial = nullptr;
        if (a.splits > 1) {
            const uint64_t at =
                (partial_row(a, b, s.start, token) * (c.kv_heads * a.group) + out_head) * a.splits + split;
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

// The (sequence, token, head) of item `at` of a workgroup's ITEMS, and the place of its
// partial results; false where there is none.
template <uint32_t ITEMS>
__device__ __forceinline__ bool item_of(const AttentionArgs &a, uint32_t heads, uint32_t at, uint32_t &head,
                                        uint64_t &row, uint64_t &partial) {
    uint32_t place = blockIdx.x, b, count = (a.upto * heads + ITEMS - 1) / ITEMS;
    if (a.starts) {
        if (!place_of(a, heads, ITEMS, place, b, count)) return false;
    } else {
        b = place / count, place %= count;
    }
    int begin, tokens, brought;
    rows_of(a, b, begin, tokens, brought);
    const uint32_t item = place * ITEMS + at, token = item / heads;
    if ((int)token >= tokens) return false;
    head = item % heads;
    row = (uint64_t)begin + token, partial = partial_row(a, b, begin, (int)token) * heads + head;
    return true;
}

// Joins the splits of one (sequence, token, head) a workgroup: the first wave
// turns the splits' maxima into weights, then D / 4 threads take a split, 1024 / D
// splits at a time. (A split without a token has sum 0 and zeros. One wave walking 64
// splits in order took 29 us after 32768 tokens, one round of memory latency a split;
// this takes 3.8.)
template <int D, bool F32>
__global__ void __launch_bounds__(256) attention_join_kernel(AttentionArgs a, uint32_t heads) {
    using T = std::conditional_t<F32, float, _Float16>;
    constexpr int ACROSS = D / 4, SIDE = 256 / ACROSS;
    __shared__ float weight[MAX_SPLITS], total;
    __shared__ __align__(16) float part[SIDE][D];
    uint32_t head;
    uint64_t row, at;
    if (!item_of<1>(a, heads, 0, head, row, at)) return;
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
        weight[tid] = w;
        if (tid == 0) total = sum;
    }
    __syncthreads();
    const uint32_t side = tid / ACROSS, x4 = 4 * (tid % ACROSS);
    const float *p = a.partial_o + at * a.splits * D + x4;
    float4 x = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (uint32_t i = side; i < a.splits; i += SIDE) {
        const float w = weight[i];
        const float4 y = *(const float4 *)(p + (uint64_t)i * D);
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

// The same where splits are few (FEW_SPLITS, 8): D / 4 threads take a (sequence, token, head) and
// walk them, four on their way together. (2 x 1000 tokens of 16 heads of 256 in three splits: the
// call takes 149 us, 160 with a workgroup each; 8 splits about even; 32 splits of one
// token 18.6, 16.3 with a workgroup each.)
template <int D, bool F32>
__global__ void __launch_bounds__(256) attention_join_rows_kernel(AttentionArgs a, uint32_t heads) {
    using T = std::conditional_t<F32, float, _Float16>;
    constexpr uint32_t ACROSS = D / 4, EACH = 4;  // splits on their way together
    const uint32_t x4 = 4 * (threadIdx.x % ACROSS);
    uint32_t head;
    uint64_t row, at;
    if (!item_of<256 / ACROSS>(a, heads, threadIdx.x / ACROSS, head, row, at)) return;
    const float *ml = a.partial_ml + 2 * at * a.splits, *p = a.partial_o + at * a.splits * D + x4;
    float4 x = make_float4(0, 0, 0, 0);
    float top = LOWEST, sum = 0.0f;
    for (uint32_t first = 0; first < a.splits; first += EACH) {
        float4 y[EACH];
        float m[EACH], l[EACH];
#pragma unroll
        for (uint32_t j = 0; j < EACH; ++j) {
            const uint32_t i = min(first + j, a.splits - 1);
            y[j] = *(const float4 *)(p + (uint64_t)i * D);
            m[j] = ml[2 * i], l[j] = ml[2 * i + 1];
            if (first + j >= a.splits) l[j] = 0.0f;
            if (l[j] == 0.0f) m[j] = LOWEST;
        }
        float above = top;
#pragma unroll
        for (uint32_t j = 0; j < EACH; ++j) above = fmaxf(above, m[j]);
        const float by = __builtin_amdgcn_exp2f(top - above);
        x.x *= by, x.y *= by, x.z *= by, x.w *= by, sum *= by, top = above;
#pragma unroll
        for (uint32_t j = 0; j < EACH; ++j) {
            const float w = l[j] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[j] - top);
            x.x += w * y[j].x, x.y += w * y[j].y, x.z += w * y[j].z, x.w += w * y[j].w, sum += w * l[j];
        }
    }
    store4((T *)a.out + row * a.out_stride + head * D + x4, x, sum == 0.0f ? 0.0f : 1.0f / sum);
}

template <int BITS, int D, int RT, bool F32>
hipError_t rows_launch(hipStream_t s, const CacheView &c, const AttentionArgs &a) {
    const uint32_t grid = (uint32_t)(c.kv_heads * a.splits * a.units);
    attention_rows_kernel<BITS, D, RT, F32><<<grid, 64 * WAVES, 0, s>>>(c, a);
    return hipGetLastError();
}

template <int BITS, int D, bool F32> hipError_t rows_rt(hipStream_t s, const CacheView &c, const AttentionArgs &a) {
    if (a.row_tiles == 1) return rows_launch<BITS, D, 1, F32>(s, c, a);
    if constexpr (D <= 128)
        if (a.row_tiles == 2) return rows_launch<BITS, D, 2, F32>(s, c, a);
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

// At least the units of all of a plan's sequences, ceil(tokens * by / of) each.
static uint64_t units_of(const AttentionArgs &a, uint64_t by, uint64_t of) {
    const uint64_t all = a.batch * ((a.upto * by + of - 1) / of);
    // sequences have more than `above` tokens, and none of them more than a unit that is not full
    const uint64_t sequences = std::min<uint64_t>(a.batch, a.rows / (a.above + 1));
    return a.starts ? std::min(all, a.rows * by / of + sequences) : all;
}
// The splits of the rows kernel's calls (plan_attention).
static uint64_t rows_splits(uint64_t groups, uint64_t reach, uint64_t cus) {
    if (reach <= 512) return 1;
    return std::max(std::min(cus / groups, (reach + 127) / 128), std::min(4 * cus / groups, (reach + 1023) / 1024));
}
// Workgroups of the kernel that joins a plan's splits: D / 4 threads a (row, head) where they are
// few, a workgroup each where they are many.
constexpr uint32_t FEW_SPLITS = 8;
static uint64_t join_groups(const AttentionArgs &a, uint32_t heads, uint32_t head_dim, uint64_t splits) {
    return units_of(a, heads, splits <= FEW_SPLITS ? 1024 / head_dim : 1);
}
// Sets the splits, as far as their partial results of `rows` query rows fit and neither kernel's
// grid passes a launch's.
static void fit_splits(uint64_t splits, uint64_t rows, uint32_t kv_heads, uint32_t heads, uint32_t head_dim,
                       uint64_t max_floats, AttentionArgs *a) {
    splits = std::min<uint64_t>(std::min<uint64_t>(splits, MAX_SPLITS), MOST_GROUPS / (kv_heads * a->units));
    splits = std::max<uint64_t>(1, splits);
    const uint64_t each = rows * heads * (head_dim + 2);
    if (splits > 1 && splits * each > max_floats) splits = std::max<uint64_t>(1, max_floats / each);
    if (splits > 1 && join_groups(*a, heads, head_dim, splits) > MOST_GROUPS) splits = 1;
    a->splits = (uint32_t)splits;
    a->floats = splits > 1 ? (splits * each + 3) / 4 * 4 : 0;  // another plan's may follow, 16-byte aligned
}

// The kernel. Few rows read the cache straight into registers; where there is enough
// work for it, a workgroup that decodes the cache once for its waves is faster:
// 48 heads of 128, F16: one prompt of 1000 tokens 39 us by rows, 46 by the prompt
// kernel; of 2000 104 and 86; 64 tokens after 8192 37 and 41, 256 tokens 100 and 87.
// The bound is on (rows x tokens they see x D) in all: 8e9, and 1.2e10 where the prompt
// kernel gains less, F32 (1000: 52 and 55; 2000: 150 and 122) and D = 64 (2000: 58 and 73;
// 3000: 116 and 104).
// The splits of the long axis, each of which costs its rows' partial outputs a
// way through memory. Rows: up to 512 tokens are one workgroup's (300 tokens: 6.6
// us, 7.7 split in three and joined); then 128 tokens each while a workgroup a CU wants
// work (4096 tokens: 8.1 us, 10.5 at 512 each), and four a CU where each has 1024
// (batch of 32 up to 16384: 83 us, 88 at two a CU, 114 at one). Prompts: where
// rows are few against the tokens they see, n that makes the least of (rounds of the workgroups that run
// at once, two a CU) / n and what joining n costs, 170 n / tokens (300 tokens
// after 16000, F16, 80 workgroups: 196 us in 3, 156 in 6, 196 in 7; 1000, 256 workgroups: 411 in
// 2, 424 in 4; a window of 4096 at D = 256, 256 workgroups: 206 in 2, 239 in 4). A prompt from its
// start on is in balance by itself (2000 tokens: 164 us split, 86 not), but for wide
// heads (4096 tokens at D = 256, 512 workgroups: 294 us, 222 in 2).
//
// A batch of both, single tokens among prompts, is two plans where its other sequences
// are short (at most 256 rows each beside the longest): up to 64 rows by rows, the
// others by the prompt kernel (a prompt of 512 among 32 single tokens after 8000: 112 us, all
// by the prompt kernel 738; two calls, which know each kind's lengths, 17 and 68).
bool plan_attention(uint32_t head_dim, uint32_t kv_heads, uint32_t f32, uint64_t max_length, uint32_t heads,
                    uint64_t max_floats, uint32_t cus, AttentionArgs *a, AttentionArgs *few) {
    max_floats = std::min<uint64_t>(max_floats, 1ull << 26);  // 256 MiB of a call's partial results
    const uint64_t rows = (uint64_t)a->max_tokens * a->group;
    uint64_t reach = max_length;  // tokens the last row and those before it may see
    if (a->window) reach = std::min<uint64_t>(reach, (uint64_t)a->window + a->max_tokens);
    const double seen = std::max((double)reach - 0.5 * a->max_tokens, 0.5 * (double)reach);
    const double work = (double)a->rows * heads * seen * head_dim;
    a->above = 0, a->upto = a->max_tokens;
    const auto tiles_of = [&](uint64_t n) { return head_dim <= 128 && n > 16 ? 2u : 1u; };
    // (the rows kernel's grid has every sequence's blocks for max_tokens; the prompt kernel's, where counts
    // differ, is sized by the rows there are)
    const uint64_t rows_groups = kv_heads * (uint64_t)a->batch * ((rows + 16 * tiles_of(rows) - 1) / (16 * tiles_of(rows)));
    a->prompt = rows > 64 && (work >= (f32 || head_dim == 64 ? 1.2e10 : 8e9) || (a->starts && rows_groups > MOST_GROUPS));
    a->row_tiles = a->prompt ? prompt_row_tiles((int)head_dim, f32) * WAVES : tiles_of(rows);
    a->blocks = (uint32_t)((rows + 16 * a->row_tiles - 1) / (16 * a->row_tiles));
    a->units = (uint64_t)a->batch * a->blocks;
    if (!a->prompt) {
        fit_splits(rows_splits((uint64_t)kv_heads * a->units, reach, cus), a->rows, kv_heads, heads, head_dim, max_floats,
                   a);
        return false;
    }
    const uint64_t others = a->rows > a->max_tokens ? a->rows - a->max_tokens : 0;  // tokens beside the longest's
    const uint32_t few_tokens = 64 / a->group;
    const bool both = a->starts && a->batch > 1 && few_tokens && others * a->group <= 256ull * (a->batch - 1);
    if (both) {
        *few = *a;
        few->prompt = 0, few->upto = few_tokens, a->above = few_tokens;
        few->row_tiles = 1;  // most bring one token
        few->blocks = (few_tokens * a->group + 15) / 16;
        few->units = (uint64_t)few->batch * few->blocks;
        fit_splits(rows_splits((uint64_t)a->batch * kv_heads, reach, cus), (uint64_t)a->batch * few_tokens, kv_heads,
                   heads, head_dim, max_floats, few);
        max_floats -= few->floats;
    }
    a->units = units_of(*a, a->group, 16 * a->row_tiles);
    // the longest's units, and the others' taken for half as long (none where they are the other plan's)
    const uint64_t others_units = both ? 0 : a->units - std::min<uint64_t>(a->units, a->blocks);
    const uint64_t busy = kv_heads * (std::min<uint64_t>(a->units, a->blocks) +
                                      (a->starts ? (others_units + 1) / 2 : others_units));
    uint64_t splits = 1;
    if (reach >= 4ull * a->max_tokens) {
        double least = 1e30;
        for (uint64_t n = 1; n <= std::max<uint64_t>(1, std::min<uint64_t>(reach / 1024, MAX_SPLITS)); ++n) {
            const double cost = (double)((busy * n + 2 * cus - 1) / (2 * cus)) / n + 170.0 * n / reach;
            if (cost < least) least = cost, splits = n;
        }
    } else if (head_dim == 256) {
        splits = std::min((cus * 5 / 2 + busy - 1) / busy, reach / 1024);
    }
    fit_splits(splits, a->rows, kv_heads, heads, head_dim, max_floats, a);
    return both;
}

// The plans of a call by themselves, on the host: for each {prompt kernel, splits, its workgroups, the
// join's (0 without one), floats of workspace, most tokens of its sequences}. Returns how many.
extern "C" int nuq_attention_plan(uint32_t head_dim, uint32_t kv_heads, uint32_t heads, uint32_t f32, uint32_t rows,
                                  uint32_t batch, uint32_t max_tokens, int ragged, uint64_t max_length, uint32_t window,
                                  uint64_t max_floats, uint32_t cus, uint64_t out[12]) {
    static const int32_t some = 0;
    AttentionArgs plans[2] = {};
    plans[0].rows = rows, plans[0].batch = batch, plans[0].max_tokens = max_tokens, plans[0].window = window;
    plans[0].group = heads / kv_heads, plans[0].starts = ragged ? &some : nullptr;
    const int count = 1 + plan_attention(head_dim, kv_heads, f32, max_length, heads, max_floats, cus, &plans[0], &plans[1]);
    for (int i = 0; i < count; ++i) {
        const AttentionArgs &a = plans[i];
        const uint64_t v[6] = {a.prompt, a.splits, kv_heads * a.splits * a.units,
                               a.splits > 1 ? join_groups(a, heads, head_dim, a.splits) : 0, a.floats, a.upto};
        std::copy(v, v + 6, out + 6 * i);
    }
    return count;
}

hipError_t launch_attention(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f32,
                            uint32_t heads, AttentionArgs a, float *work) {
    if (a.splits > 1) {
        a.partial_o = work;
        a.partial_ml = work + a.floats / (head_dim + 2) * head_dim;
    }
    const hipError_t e = a.prompt ? launch_attention_prompt(s, c, bits, head_dim, f32, a)
                         : f32    ? rows_dispatch<true>(s, c, bits, head_dim, a)
                                  : rows_dispatch<false>(s, c, bits, head_dim, a);
    if (e != hipSuccess || a.splits == 1) return e;
    const bool few_splits = a.splits <= FEW_SPLITS;
    const uint32_t grid = (uint32_t)join_groups(a, heads, head_dim, a.splits);
#define NUQ_CASE(D)                                                                             \
    if (head_dim == D) {                                                                        \
        if (few_splits && f32) attention_join_rows_kernel<D, true><<<grid, 256, 0, s>>>(a, heads); \
        else if (few_splits) attention_join_rows_kernel<D, false><<<grid, 256, 0, s>>>(a, heads);  \
        else if (f32) attention_join_kernel<D, true><<<grid, 256, 0, s>>>(a, heads);            \
        else attention_join_kernel<D, false><<<grid, 256, 0, s>>>(a, heads);                    \
    }
    NUQ_CASE(64) NUQ_CASE(128) NUQ_CASE(256)
#undef NUQ_CASE
    return hipGetLastError();
}

}  // namespace nuq
