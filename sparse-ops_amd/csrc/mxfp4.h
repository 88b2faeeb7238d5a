// Microscaled 4-bit floating point: blocks of 32 entries along the contraction, each entry one of +-{0, .5, 1, 1.5, 2, 3, 4, 6} (codes 0..7, +8 for minus), the
// block's scale 2^(s - 127) in a byte s (255: not a number).
//
// Outside, row-major: 16 bytes of codes a block, the even entry of two in the low half of a byte; scales beside.
// Inside, as the scaled matrix instruction (16 x 16 x 128) takes an operand, lane l holding row l % 16 and block l / 16 of four: tiles of 32 rows, in a tile unit by unit of 8
// blocks, of a unit four operands of 64 lanes x 16 bytes: the first four blocks of rows 0..15, of rows 16..31, the last four of both.  A unit's scales are one word a lane, a byte
// for each operand: lane l, byte 2 * (row / 16) + (block / 4) for row % 16 = l % 16, block % 4 = l / 16.  Blocks are padded to whole units with zeros.
#pragma once
#include "elements.h"
#include "so_internal.h"

constexpr uint32_t kMxTile = 32;        // rows of a tile
constexpr uint32_t kMxUnit = 8;         // blocks that share a word of scales
constexpr uint32_t kMxZero = 127;       // the scale of padding: 2^0, so that it adds zeros

typedef uint32_t so_u32x4 __attribute__((ext_vector_type(4)));

struct so_mxfp4 {
    uint32_t m = 0, n = 0;
    uint32_t blocks = 0;                // of a row as stored, a multiple of kMxUnit
    uint32_t tiles = 0;
    int device = 0;
    void *d_blob = nullptr;             // one allocation for the two
    so_u32x4 *d_codes = nullptr;        // [tiles][units][4][64]
    uint32_t *d_scales = nullptr;       // [tiles][units][64]
};

// Where the codes (by 16 bytes) and the scale (by bytes) of block b of a row lie.
__host__ __device__ inline uint64_t so_mx_code_at(uint64_t row, uint32_t b, uint32_t units)
{
    return ((row / kMxTile * units + b / kMxUnit) * 4u + b % kMxUnit / 4u * 2u + row % kMxTile / 16u) * 64u + b % 4u * 16u + row % 16u;
}
__host__ __device__ inline uint64_t so_mx_scale_at(uint64_t row, uint32_t b, uint32_t units)
{
    return ((row / kMxTile * units + b / kMxUnit) * 64u + b % 4u * 16u + row % 16u) * 4u + row % kMxTile / 16u * 2u + b % kMxUnit / 4u;
}

static inline uint32_t so_mx_blocks(uint32_t n) { return so_ceil_div(n, 32 * kMxUnit) * kMxUnit; }

// The scale of a block whose largest magnitude has these bits (fp32 without its sign).  2^(floor(log2) - 2), so that the largest entry lands in 4..8, at least 2^-127.
__device__ __forceinline__ uint32_t so_mx_scale(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : max(e, 2u) - 2u;
}

// 2^(s - 127) for s < 255, exactly: s = 0 is a subnormal number.
__device__ __forceinline__ float so_mx_power(uint32_t s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

// Eight entries as codes in a word, the first in the lowest bits: nearest, ties to the even code, beyond 6 to 6 (v_cvt_scalef32_pk_fp4_f32).
__device__ __forceinline__ uint32_t so_mx_codes(const float (&v)[8], float scale)
{
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    return w;
}

// csrc/mxfp4.hip: X [n x C] quantised in blocks of 32 of its rows, into tiles of 32 columns as above.  Without `codes` only whether it is small enough for a launch.
so_status so_mx_quantize_columns(so_ctx *ctx, int type, const void *dX, size_t x_stride, uint32_t n, uint32_t C, so_u32x4 *codes, uint32_t *scales);
