// Byte layout of the quantised paged K/V cache (include/nuq.h, nuq_cache),
// shared by the kernels that write, read and attend to it.
//
// A cache is [pages][kv heads][page_tokens / 16] tiles. A tile holds 16
// tokens of one head: K codes, K scales, V codes, V scales. Values come in
// groups of 32 along the head dimension D with one f16 scale d each:
//   4 bits: m = the group's value of largest magnitude (the positive one on a
//           tie), d = f16(bf16(clamp(-m / 8, +-2720))), code = clamp(rint(x / d), -8, 7)
//   8 bits: d = f16(min(up4(max|x| / 127), 56)), up4 the next value of 4
//           significant bits, code = clamp(rint(x / d), -127, 127)
// stored with an offset of 8 (128). The value is d * code. d has 8 (4)
// significant bits, so d * code (8 + 3 bits; -8 is a power of two; 4 + 7) is an
// f16 number exactly, and so is the bias 24 d (1152 d) below: a code becomes
// its value by one f16 fma without a rounding, and the limits on d keep the
// bias finite (24 * 2720 and 1152 * 56 are below 65504). Where d is below
// f16's normal range all of these are multiples of 2^-24, exact too.
//
// The two planes are laid out so that one lane's wide load is its operand of
// v_mfma_f32_16x16x32_f16 (lane l: row l % 16, k = 8 * (l / 16) ..):
//   K codes  [unit][token 16][quarter 4][chunk]: k runs along D, so the lane of
//            token n and quarter h reads, for every group of the unit, the
//            dimensions 32 g + 8 h ..+7: one word at 4 bits (dimension 2 p at bit
//            4 p, 2 p + 1 at bit 16 + 4 p, so one mask takes a pair), 8 bytes at 8
//   K scales [token 16][group]
//   V codes  [unit][quad 4][column 16][token of the quad 4][chunk / 4]: k runs
//            along tokens, so the lane of column n and quad h reads four tokens'
//            codes of its D / units / 16 consecutive dimensions (dimension j at
//            bit 4 j or byte j); a token's own codes never share a byte with another's
//   V scales [quad 4][group][token of the quad 4]
// A unit is what one chunk (at most 16 bytes a lane) covers: 128 dimensions at
// 4 bits (64 where D is 64), 64 at 8 bits.
//
// A token-head whose K or V held a non-finite value is stored with NaN K scales
// and zero V scales: it reads back as NaN, and makes NaN the rows that
// attend to it and no others (masked scores are replaced before the softmax,
// while a NaN in V would reach masked rows as 0 * NaN).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nuq {

template <int BITS, int D> struct CacheGeometry {
    static constexpr int GROUPS = D / 32;
    static constexpr int CHUNK = D * BITS / 32 < 16 ? D * BITS / 32 : 16;  // bytes a lane loads of a unit
    static constexpr int UNITS = D * BITS / 32 / CHUNK;
    static constexpr int UNIT_DIMS = D / UNITS;
    static constexpr int UNIT_GROUPS = UNIT_DIMS / 32;
    static constexpr int COLUMN = UNIT_DIMS / 16;  // consecutive dimensions of a V column
    static constexpr int CODES = 2 * D * BITS;     // bytes of a plane's codes in a tile
    static constexpr int SCALES = D;               // 16 tokens * D / 32 groups * 2 bytes
    static constexpr int K_SCALES = CODES, V_CODES = CODES + SCALES, V_SCALES = 2 * CODES + SCALES;
    static constexpr int TILE_BYTES = 2 * (CODES + SCALES);
    static constexpr int OFFSET = BITS == 4 ? 8 : 128;
};

// What the kernels need of a nuq_cache.
struct CacheView {
    uint8_t *bytes;
    uint32_t pages;
    uint32_t kv_heads;
    uint32_t tiles_log2;  // log2 of the tiles in a page
};

}  // namespace nuq
