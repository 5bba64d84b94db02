// mx_common.hpp -- microscaled rows (dr_mx_rows), shared by mx_rows.hip
// (quantisation, norm) and the products of mx_ring.hip and mx_tile.hip.
//
// 32 consecutive values of a row are a block: they share 2^e, held as the byte
// e + 127 (255: the whole block stands for NaN), and each is an E2M1 (4 bit) or
// E4M3 (8 bit) code times 2^e.  With a = max |x| of the block, e is the smallest
// that keeps a / 2^e within the largest code (6 or 448), so nothing saturates;
// e >= -126, which keeps 2^-e a normal f32 number (blocks of zeros have e = -126).
// Codes are to nearest, ties to even.
//   codes   [n][cols / 2] bytes (value 2 j in the low half of byte j), or [n][cols]
//   scales  [n][mx_pitch(cols)]: one byte per block, rows at multiples of 4 bytes
//           so that four blocks' bytes are one aligned load; the bytes between
//           a row's last block and the next row are neither read as scales nor
//           written.
#pragma once

#include <type_traits>

#include "dr_internal.hpp"

namespace dr {
namespace {

constexpr int MX_NAN = 255;

using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using bf16x8m = __bf16 __attribute__((ext_vector_type(8)));
using f32x2m = float __attribute__((ext_vector_type(2)));
using f32x4m = float __attribute__((ext_vector_type(4)));
using u32x4m = uint32_t __attribute__((ext_vector_type(4)));
using u32x2m = uint32_t __attribute__((ext_vector_type(2)));

// Scale byte of a block whose largest magnitude has the bit pattern `bits` (sign
// cleared; compared as integers, so a NaN is larger than an infinity, and that
// larger than every number).
template <int FMT>
__device__ __forceinline__ int mx_scale_byte(uint32_t bits) {
    if (bits >= 0x7f800000u) return MX_NAN;
    const int top = FMT == MX_E2M1 ? 2 : 8;
    const uint32_t frac = FMT == MX_E2M1 ? 0x400000u : 0x600000u;  // of 6 = 1.5 * 2^2 and 448 = 1.75 * 2^8
    const int e = (int)(bits >> 23) - top + ((bits & 0x7fffffu) > frac ? 1 : 0);
    return e < 1 ? 1 : e;
}

// 2^e of a scale byte as f32, NaN for MX_NAN.
__device__ __forceinline__ float mx_scale(int byte) {
    return __uint_as_float(byte == 0 ? 0x400000u : byte == MX_NAN ? 0x7fc00000u : (uint32_t)byte << 23);
}

// The codes of 8 values with their block's scale byte: 4 bytes (E2M1) or 8.
// Dividing by a power of two is exact but for results far below the smallest code.
template <int FMT>
__device__ __forceinline__ u32x2m mx_encode8(const float (&x)[8], int byte) {
    u32x2m c = {0, 0};
    if (byte == MX_NAN) return c;
    if constexpr (FMT == MX_E2M1) {
        const float s = __uint_as_float((uint32_t)byte << 23);
        c[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[0], x[0], x[1], s, 0);
        c[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[0], x[2], x[3], s, 1);
        c[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[0], x[4], x[5], s, 2);
        c[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[0], x[6], x[7], s, 3);
    } else {
        const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * inv, x[4 * h + 1] * inv, 0, false);
            c[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * inv, x[4 * h + 3] * inv, w, true);
        }
    }
    return c;
}

// The f32 values of 8 codes.
template <int FMT>
__device__ __forceinline__ void mx_decode8(u32x2m c, int byte, float (&x)[8]) {
    const float s = mx_scale(byte);
    f32x2m p[4];
    if constexpr (FMT == MX_E2M1) {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], 1.0f, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], 1.0f, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], 1.0f, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], 1.0f, 3);
    } else {
        p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[0], false);
        p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[0], true);
        p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[1], false);
        p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[1], true);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i / 2][i % 2] * s;
}

// The codes of 4 values: 2 bytes (E2M1) or 4.
template <int FMT>
__device__ __forceinline__ uint32_t mx_encode4(const float (&x)[4], int byte) {
    if (byte == MX_NAN) return 0;
    if constexpr (FMT == MX_E2M1) {
        const float s = __uint_as_float((uint32_t)byte << 23);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, x[0], x[1], s, 0), x[2], x[3], s, 1);
    } else {
        const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, w, true);
    }
}

// The largest of a value over a quad of lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));  // lanes 1 0 3 2
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));  // lanes 2 3 0 1
}

__device__ __forceinline__ uint16_t mx_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float mx_f32(uint32_t bf16_bits) { return __uint_as_float(bf16_bits << 16); }

// 8 consecutive f32 or bf16 values (16-byte aligned).
template <bool BF16>
__device__ __forceinline__ void load8(const void* base, size_t at, float (&x)[8]) {
    if constexpr (BF16) {
        const u32x4m v = *reinterpret_cast<const u32x4m*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = mx_f32(v[i] & 0xffff), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    } else {
        const f32x4m* p = reinterpret_cast<const f32x4m*>(static_cast<const float*>(base) + at);
        const f32x4m a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    }
}
template <bool BF16>
__device__ __forceinline__ void store8(void* base, size_t at, const float (&x)[8]) {
    if constexpr (BF16) {
        u32x4m v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = mx_bf16(x[2 * i]) | (uint32_t)mx_bf16(x[2 * i + 1]) << 16;
        *reinterpret_cast<u32x4m*>(static_cast<uint16_t*>(base) + at) = v;
    } else {
        f32x4m* p = reinterpret_cast<f32x4m*>(static_cast<float*>(base) + at);
        p[0] = f32x4m{x[0], x[1], x[2], x[3]};
        p[1] = f32x4m{x[4], x[5], x[6], x[7]};
    }
}

// x / (1 + e^-x), and gelu in its tanh form: 0.5 x (1 + tanh z) = x / (1 + e^-2z),
// z = sqrt(2 / pi) (x + 0.044715 x^3), which keeps its digits where tanh is near -1.
__device__ __forceinline__ float mx_act(float x, int fn) {
    const float z = fn == MX_SILU ? x : 1.5957691216057308f * (x + 0.044715f * x * x * x);
    return x / (1.0f + expf(-z));
}

// f(Int<0>{}) .. f(Int<N - 1>{})
template <int I>
using Int = std::integral_constant<int, I>;
template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(Int<I>{});
        static_for<N, I + 1>(f);
    }
}

// ---- staging through LDS (mx_ring.hip, mx_tile.hip)

using i32x8m = int __attribute__((ext_vector_type(8)));

// The block-scaled MFMA adds 8 consecutive columns' products as numbers of fixed point, whose
// last bit is 2^-13 of the power of two of the largest: what a smaller product has below
// it is dropped.  Eights are then added in f32.  E2M1 codes' products span 2^5 and are a multiple of
// 2^-2, so nothing is dropped.  E4M3 codes go through in two parts that keep theirs too: those
// of 2 and more (bit 6; products of 2^10 to a multiple of 2^-3) and those below
// (of 2^2 to a multiple of 2^-10), with 0 in the others' places.  Random codes and blocks: each part's
// sums equal the exact ones; in one part they are off by up to 1e-4 of the sum of magnitudes.
__device__ __forceinline__ void mx_split(const i32x8m& c, i32x8m& large, i32x8m& small) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = (uint32_t)c[i] >> 6 & 0x01010101u;
        large[i] = c[i] & (int)((b << 8) - b);
        small[i] = c[i] ^ large[i];
    }
}

constexpr int OUT_OF_RANGE = 1 << 30;  // at or past every tile's end (256 rows of 2^22 bytes at most)

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base, size_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
// lane i: 16 (4) bytes at rsrc + voff + soff -> LDS byte address lds + 16 (4) i; 0 where voff
// lies past the buffer's end (dword by dword; the range check leaves soff out, so a lane whose
// own bytes may end before voff + soff + 16 must not ask).  Inline asm without outputs, so that the compiler does not
// make every LDS read wait for it; the kernels' own waits order them.  (M0 needs a wait
// state; nothing else here uses it.)
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t lds, int voff, int soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(r), "s"(soff)
                 : "memory");
#endif
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, uint32_t lds, int voff, int soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(r), "s"(soff)
                 : "memory");
#endif
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// this wave's LDS reads and writes are done
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// a barrier that leaves LDS DMA in flight
__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}

// Place in the order of tiles of workgroup id of `total`: workgroups go to the 8 XCDs
// in turn, and each XCD takes a run of consecutive places, whose operands its L2 shares.
__device__ __forceinline__ int xcd_order(int id, int total) {
    const int x = id & 7, per = total >> 3, rest = total & 7;
    return x * per + min(x, rest) + (id >> 3);
}

// 16-byte piece c of row R of a staged tile lies at slot c ^ turn(R), so that a read of
// one piece per lane group of 16 rows, or (PAIRS, 128-byte rows) of one of two that
// belong together, touches every bank once (a read serves lanes 0-3, 12-15 and 20-27 at a
// time, so rows 0-3 and 12-15 of a group meet rows 4-11 of the next): SQ_LDS_BANK_CONFLICT is 0
// in the tiles' kernels.  The ring kernels have some: where 4 activation rows are staged, two of
// them meet in a bank (16 cycles of a step's 48 of LDS; loads bound it), and the sums are
// written over rows of 20 floats.  ROW: bytes of a row, 64, 128 or more.
template <int ROW, bool PAIRS = false>
__device__ __forceinline__ int turn(int R) {
    if (ROW == 64) return (R >> 1) & 3;
    if (ROW == 128 && PAIRS) return (((R >> 2) ^ (R >> 3)) & 1) | (R & 2) | ((R & 8) >> 1);
    return ROW == 128 ? (R >> 1) & 7 : R & 15;
}

// One sum of a product, with its residual, at element `at` of out.
__device__ __forceinline__ void put_sum(const MxMatArgs& a, size_t at, float x) {
    if (a.bf16) {
        if (a.residual) x += mx_f32(static_cast<const uint16_t*>(a.residual)[at]);
        static_cast<uint16_t*>(a.out)[at] = mx_bf16(x);
    } else {
        if (a.residual) x += static_cast<const float*>(a.residual)[at];
        static_cast<float*>(a.out)[at] = x;
    }
}

}  // namespace
}  // namespace dr
