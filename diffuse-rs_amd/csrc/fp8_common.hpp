// fp8_common.hpp -- the 8 bit cache format (DR_PRECISION_FP8 layers), shared by
// kv_fp8.hip (store, gather) and attn_fp8.hip (attention).
//
// A block is one position of one KV head: its head_dim values share a power of
// two 2^e and are held as e4m3 codes (x / 2^e to nearest, ties to even).  With
// a = max |x|: e = floor(log2 a) - 8, one more where a's mantissa exceeds 1.75,
// so a / 2^e <= 448, the largest e4m3 value, and nothing saturates; e >= -126.
// The scale byte is e + 127; 0 is a row of zeros, stored or never stored, so that
// 1 and above always mean values; FP8_NAN marks a row with a NaN or an infinity,
// which has no 8 bit form: its codes are 0 and all of it reads back as NaN.
// The block is a single position because a denoise step rewrites single
// positions: a scale shared by more of them would make each store read and
// requantise its neighbours, and the contents depend on the order of stores.
//
// Planes of a layer and batch slot, per KV head and 32-position tile (HD: the
// head-dim tile; a tile of either plane is one contiguous block of 32 * HD
// bytes, in the order in which the attention's MFMA operands take it):
//   K   [n_head_kv][cap / 32][HD / 16][32][16]   16-value chunk, position, value
//   V   [n_head_kv][cap / 32][HD][32]            value, position
//   scale bytes [n_head_kv][cap / 32][2][32]     K's, then V's: one 64-byte line
#pragma once

#include "dr_internal.hpp"

namespace dr {
namespace {

constexpr int FP8_NAN = 255;

// Scale byte of a row whose largest magnitude has the bit pattern `bits` (sign
// cleared; compared as integers, so a NaN is larger than an infinity, and that
// larger than every number).
__device__ __forceinline__ int fp8_scale_byte(uint32_t bits) {
    if (bits >= 0x7f800000u) return FP8_NAN;
    if (bits == 0) return 0;
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}

// 2^-e of a scale byte (0..247): x times it is exact but for results far below
// the smallest code.
__device__ __forceinline__ float fp8_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// 2^e of a scale byte: 0 for byte 0 and infinity for FP8_NAN, whose codes are
// all 0 (so their products are 0 and NaN).
__device__ __forceinline__ float fp8_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Byte offsets of a tile (t = position / 32) of KV head g.
__device__ __forceinline__ size_t fp8_tile(int g, int cap, int t, int hd_tile) {
    return ((size_t)g * (cap / 32) + t) * 32 * hd_tile;
}
__device__ __forceinline__ size_t fp8_scale_tile(int g, int cap, int t) {
    return ((size_t)g * (cap / 32) + t) * 64;
}

}  // namespace
}  // namespace dr
